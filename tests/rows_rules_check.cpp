// Evaluates the launch rules of the operators between two attention blocks (gemma4-webgpu_amd/csrc/launch_rules.h) for
// tests/test_rows_rules.py: reads "<rule> <arguments>" lines and prints one value a line.
#include <stdio.h>

#include <iostream>
#include <string>

#include "../gemma4-webgpu_amd/csrc/launch_rules.h"

int main() {
    std::string rule;
    while (std::cin >> rule) {
        uint32_t a = 0, b = 0, d = 0;
        uint64_t c = 0;
        if (rule == "long_row_columns" && std::cin >> a)
            printf("%u\n", g4::long_row_columns(a));
        else if (rule == "linear8_tile" && std::cin >> a >> b >> c >> d)
            printf("%u\n", g4::linear8_tile(a, b, c, d));
        else
            return fprintf(stderr, "unknown rule %s\n", rule.c_str()), 1;
    }
    return 0;
}
