"""Argument checks of the operators between two attention blocks on the CPU: refused on the host, with a message, before
anything is enqueued; struct layouts; workspace sizes."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from g4attn import abi, ops

HEADER = Path(__file__).resolve().parent.parent / "include" / "g4attn.h"
STRUCTS = {"g4_add_rms_norm_params": abi.AddRmsNormParams, "g4_quantize_rows_params": abi.QuantizeRowsParams,
           "g4_lora": abi.Lora, "g4_linear_e4m3_params": abi.LinearE4m3Params, "g4_lora_add_params": abi.LoraAddParams}


def test_struct_layouts_match_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} __sizeof__ %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, *_ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    for line in out.split("\n"):
        if line:
            cname, field, value = line.split()
            py = STRUCTS[cname]
            assert int(value) == (C.sizeof(py) if field == "__sizeof__" else getattr(py, field).offset), line


def refused(status, want, code=abi.G4_EINVAL):
    msg = abi.load().g4_last_error().decode()
    assert status == code and want in msg, (status, msg)


def norm(x=256, residual=512, post=None, weight=1024, total=2048, out=4096, scales=8192, **kw):
    p = dict(rows=4, n=64, x_type=0, residual_type=0, weight_type=1, out_type=3, eps=1e-6, reserved=0, x_stride=0,
             residual_stride=0, residual_out_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_add_rms_norm(x, residual, post, weight, total, out, scales, abi.AddRmsNormParams(**p), None)


@pytest.mark.parametrize("args,want", [
    (dict(rows=(1 << 22) + 1), "rows"), (dict(n=0), "n 0"), (dict(n=32769), "n 32769"), (dict(x_type=3), "x_type 3"),
    (dict(residual_type=3), "residual_type 3"), (dict(weight_type=3), "weight_type"), (dict(out_type=4), "out_type 4"),
    (dict(reserved=1), "reserved"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=None), "NULL x"),
    (dict(out=None, total=None, weight=None, scales=None), "neither"), (dict(out=None, scales=None), "weight without out"),
    (dict(scales=None), "scales"), (dict(out_type=0), "scales"), (dict(out=None, weight=None), "scales"),
    (dict(x_stride=63), "x_stride"), (dict(residual_stride=1), "residual_stride"), (dict(out_stride=63), "out_stride"),
    (dict(residual_out_stride=(1 << 40) + 1), "residual_out_stride"), (dict(x=258), "misaligned x"),
    (dict(residual=514), "misaligned residual"), (dict(weight=1025), "misaligned weight"), (dict(scales=8194), "misaligned scales"),
])
def test_add_rms_norm_refuses(args, want):
    refused(norm(**args), want)


def test_no_rows_is_no_call():
    assert norm(rows=0) == abi.G4_OK
    p = abi.QuantizeRowsParams(0, 64, 0, 0, 0, 0)
    assert abi.load().g4_quantize_rows(256, 512, 1024, p, None) == abi.G4_OK
    assert abi.load().g4_add_rms_norm(256, None, None, None, 512, None, None, None, None) == abi.G4_EINVAL


@pytest.mark.parametrize("ptrs,params,want", [
    ((None, 512, 1024), {}, "NULL"), ((256, None, 1024), {}, "NULL"), ((256, 512, None), {}, "NULL"),
    ((256, 512, 1024), dict(x_type=3), "x_type 3"), ((256, 512, 1024), dict(n=0), "n 0"),
    ((256, 512, 1024), dict(rows=1 << 23), "rows"), ((256, 512, 1024), dict(reserved=2), "reserved"),
    ((256, 512, 1024), dict(x_stride=3), "x_stride"), ((256, 512, 1024), dict(out_stride=3), "out_stride"),
    ((257, 512, 1024), {}, "misaligned x"), ((256, 512, 1025), {}, "misaligned scales"),
])
def test_quantize_rows_refuses(ptrs, params, want):
    p = dict(rows=4, n=64, x_type=0, reserved=0, x_stride=0, out_stride=0)
    p.update(params)
    refused(abi.load().g4_quantize_rows(*ptrs, abi.QuantizeRowsParams(**p), None), want)


def lora(**kw):
    p = dict(a=4096, b=8192, scales=256, n_adapters=4, rank=16, n=64, n_segs=2, widths=(C.c_uint32 * 4)(40, 24, 0, 0), type=1,
             reserved=0)
    p.update(kw)
    return abi.Lora(**p)


LORA = [
    (dict(a=None), "NULL adapters"), (dict(b=None), "NULL adapters"), (dict(a=4104), "16-byte aligned"), (dict(b=8200), "16-byte aligned"),
    (dict(scales=255), "scales"), (dict(n_adapters=0), "0 adapters"), (dict(n_adapters=65536), "65536 adapters"),
    (dict(rank=0), "rank 0"), (dict(rank=12), "rank 12"), (dict(rank=136), "rank 136"), (dict(n=0), "n 0"), (dict(n=72), "n 72"),
    (dict(n=65552), "n 65552"), (dict(n_segs=0), "0 segments"), (dict(n_segs=5), "5 segments"), (dict(type=0), "adapter type 0"),
    (dict(type=3), "adapter type 3"), (dict(reserved=1), "reserved"), (dict(n_segs=3), "segment 2 has no outputs"),
    (dict(widths=(C.c_uint32 * 4)(1 << 20, 1, 0, 0)), "outputs"),
    (dict(widths=(C.c_uint32 * 4)((1 << 32) - 1, (1 << 32) - 1, 0, 0)), "outputs"),
]


def linear(low=None, ids=None, x=256, xs=256, w=256, ws=256, out=256, space=256, size=1 << 40, **kw):
    p = dict(n_tokens=4, rows=64, n=64, out_type=0, x_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_linear_e4m3(x, xs, w, ws, low, ids, out, abi.LinearE4m3Params(**p), space, size, None)


def lora_add(low, ids=256, x=256, xs=None, base=256, out=256, space=256, size=1 << 40, **kw):
    p = dict(n_tokens=4, x_type=1, out_type=0, reserved=0, x_stride=0, base_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_lora_add(low, ids, x, xs, base, out, abi.LoraAddParams(**p), space, size, None)


@pytest.mark.parametrize("args,want", LORA)
def test_adapters_are_checked_by_every_entry_point(args, want):
    n = C.c_size_t(0)
    refused(linear(lora(**args), 256), want)
    refused(lora_add(lora(**args)), want)
    refused(abi.load().g4_lora_workspace_size(lora(**args), 4, C.byref(n)), want)
    p = abi.LinearE4m3Params(4, 64, 64, 0, 0, 0)
    refused(abi.load().g4_linear_e4m3_workspace_size(p, lora(**args), C.byref(n)), want)


@pytest.mark.parametrize("args,want", [
    (dict(n_tokens=(1 << 22) + 1), "tokens"), (dict(rows=0), "0 rows"), (dict(rows=(1 << 20) + 1), "rows"), (dict(n=0), "n 0"),
    (dict(n=24), "n 24"), (dict(n=1 << 17), "n 131072"), (dict(out_type=3), "out_type 3"), (dict(x_stride=48), "x_stride"),
    (dict(out_stride=63), "out_stride"), (dict(x_stride=72), "16-byte aligned"), (dict(x=264), "16-byte aligned"),
    (dict(w=264), "16-byte aligned"), (dict(x=None), "NULL"), (dict(xs=None), "NULL"), (dict(w=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(out=None), "NULL"), (dict(space=None), "NULL"), (dict(out=258), "misaligned"), (dict(xs=258), "misaligned"),
    (dict(space=264), "workspace must be"), (dict(low=lora()), "go together"), (dict(ids=256), "go together"),
    (dict(low=lora(), ids=256, n=128), "beside a projection"), (dict(low=lora(), ids=256, rows=65), "beside a projection"),
    (dict(x_stride=(1 << 40) + 16), "too long"),
])
def test_linear_e4m3_refuses(args, want):
    refused(linear(**args), want)


def test_linear_e4m3_workspace():
    refused(linear(lora(), 256, size=64), "workspace", abi.G4_ENOSPC)
    assert linear(n_tokens=0) == abi.G4_OK and linear(lora(), 256, n_tokens=0) == abi.G4_OK
    refused(abi.load().g4_linear_e4m3_workspace_size(abi.LinearE4m3Params(4, 64, 64, 0, 0, 0), None, None), "bytes is NULL")


@pytest.mark.parametrize("args,want", [
    (dict(n_tokens=1 << 23), "tokens"), (dict(x_type=4), "x_type 4"), (dict(out_type=3), "out_type 3"), (dict(reserved=1), "reserved"),
    (dict(ids=None), "NULL"), (dict(x=None), "NULL"), (dict(base=None), "NULL"), (dict(out=None), "NULL"), (dict(space=None), "NULL"),
    (dict(xs=256), "x_scales"), (dict(x_type=3), "x_scales"), (dict(x_stride=63), "stride"), (dict(base_stride=63), "stride"),
    (dict(out_stride=63), "stride"), (dict(x=264), "16-byte aligned"), (dict(x_stride=68), "16-byte aligned"),
    (dict(base=258), "misaligned"), (dict(out=258), "misaligned"), (dict(ids=258), "misaligned"), (dict(space=264), "workspace must be"),
    (dict(out_stride=(1 << 40) + 1), "too long"),
])
def test_lora_add_refuses(args, want):
    refused(lora_add(lora(), **args), want)


def test_lora_add_workspace():
    refused(lora_add(lora(), size=64), "workspace", abi.G4_ENOSPC)
    refused(lora_add(None), "NULL lora")
    assert lora_add(lora(), n_tokens=0) == abi.G4_OK
    refused(abi.load().g4_lora_workspace_size(lora(), 1 << 23, C.byref(C.c_size_t(0))), "tokens")


@pytest.mark.parametrize("rank,n,rows", [(16, 1536, 2560), (128, 64, 96), (8, 8192, 1536)])
def test_a_workspace_serves_every_smaller_call(rank, n, rows):
    """The size never falls with the tokens, and a call of fewer tokens needs no more (refused before the launch if it did)."""
    low = lora(rank=rank, n=n, n_segs=1, widths=(C.c_uint32 * 4)(rows, 0, 0, 0))
    last = [0, 0, 0]
    for tokens in [1, 2, 15, 16, 17, 64, 65, 255, 256, 257, 500, 1000, 2048, 3000, 4096, 5000, 16384, 100000]:
        p = abi.LinearE4m3Params(tokens, rows, n, 0, 0, 0)
        sizes = []
        for call in (lambda b: abi.load().g4_lora_workspace_size(low, tokens, b),
                     lambda b: abi.load().g4_linear_e4m3_workspace_size(p, low, b),
                     lambda b: abi.load().g4_linear_e4m3_workspace_size(p, None, b)):
            b = C.c_size_t(0)
            assert call(C.byref(b)) == abi.G4_OK
            sizes.append(b.value)
        assert all(s >= m for s, m in zip(sizes, last)), (tokens, sizes, last)
        last = sizes


@pytest.mark.parametrize("args,want", [
    (dict(out=256), "out and x"), (dict(out=256, out_type=0, scales=None, out_stride=80), "out and x"), (dict(out=2048), "out is"),
    (dict(out=512), "out and residual"), (dict(total=256, residual_type=1), "residual_out and x"),
    (dict(total=512, residual_stride=72), "residual_out and residual"), (dict(total=256, x_stride=72), "residual_out and x"),
])
def test_add_rms_norm_refuses_to_share_memory_with_other_rows(args, want):
    refused(norm(**args), want)


def test_quantize_rows_and_lora_add_refuse_to_share_memory_with_other_rows():
    lib = abi.load()
    refused(lib.g4_quantize_rows(256, 256, 1024, abi.QuantizeRowsParams(4, 64, 0, 0, 0, 0), None), "out is x")
    refused(lib.g4_lora_add(lora(), 256, 4096, None, 512, 512, abi.LoraAddParams(4, 0, 0, 0, 0, 0, 80), 4096, 1 << 20, None),
            "base may be out")


def test_python_wrappers_refuse_tensors_of_the_cpu():
    x, w = torch.zeros(2, 64), torch.zeros(64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        ops.add_rms_norm(x, w, torch.zeros(2, 64))
    with pytest.raises(ValueError, match="GPU"):
        ops.quantize_rows(x, x, w)
    with pytest.raises(TypeError, match="expected a tensor"):
        ops.quantize_rows(None, x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_e4m3(x, w, x, w, x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.LoraAdapters(torch.zeros(2, 8, 64, dtype=torch.float16), torch.zeros(2, 64, 8, dtype=torch.float16))


@pytest.mark.parametrize("kind", [abi.G4_F32, abi.G4_F16, abi.G4_BF16])
def test_sums_in_f32_go_with_every_output_type_and_nothing_else_does(kind):
    assert linear(out_type=kind | abi.G4_F32_SUMS, n_tokens=0) == abi.G4_OK
    refused(linear(out_type=abi.G4_E4M3 | abi.G4_F32_SUMS), "out_type")
    for other in (kind | 0x200, kind | 0x80, kind | 0x80000000, kind | abi.G4_F32_SUMS | 0x10):
        refused(linear(out_type=other), "out_type")
    header = HEADER.read_text()
    assert f"#define G4_F32_SUMS {abi.G4_F32_SUMS:#x}" in header
