"""Argument checks of the paged-cache and log-probability entry points on the CPU: refused on the host, with a message,
before anything is enqueued; struct layouts; workspace sizes."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from g4attn import abi, ops

HEADER = Path(__file__).resolve().parent.parent / "include" / "g4attn.h"
STRUCTS = {"g4_paged_cache": abi.PagedCache, "g4_paged_batch": abi.PagedBatch,
           "g4_paged_append_params": abi.PagedAppendParams, "g4_paged_attn_params": abi.PagedAttnParams,
           "g4_token_logprobs_params": abi.TokenLogprobsParams}


def test_struct_layouts_match_c(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} __sizeof__ %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout
    for line in out.split("\n"):
        if line:
            cname, field, value = line.split()
            py = STRUCTS[cname]
            assert int(value) == (C.sizeof(py) if field == "__sizeof__" else getattr(py, field).offset), line


def cache(**kw):
    d = dict(k_pool=4096, v_pool=8192, num_pages=100, page_size=64, num_kv_heads=1, head_dim=256, dtype=0, reserved=0)
    d.update(kw)
    return abi.PagedCache(**d)


def batch(**kw):
    d = dict(block_table=64, token_start=64, ctx_lens=64, positions=None, tree_mask=None, n_seqs=4, table_stride=10,
             n_tokens=32, max_tokens=8, mask_words=0, reserved=0)
    d.update(kw)
    return abi.PagedBatch(**d)


def attn(c, b, q=256, out=256, nqh=8, window=0, scale=1.0, cap=0.0, ws=256, size=1 << 40):
    lib = abi.load()
    st = lib.g4_paged_attn(c, b, q, out, abi.PagedAttnParams(nqh, window, scale, cap), ws, size, None)
    return st, lib.g4_last_error().decode()


SHARED = [
    (dict(head_dim=128), {}, "head_dim 128"), (dict(head_dim=0), {}, "head_dim 0"),
    (dict(page_size=8), {}, "page_size 8"), (dict(page_size=48), {}, "page_size 48"), (dict(page_size=2048), {}, "page_size"),
    (dict(page_size=0), {}, "page_size 0"), (dict(dtype=2), {}, "dtype 2"), (dict(num_kv_heads=0), {}, "num_kv_heads 0"),
    (dict(num_kv_heads=5000), {}, "num_kv_heads"), (dict(num_pages=0), {}, "num_pages 0"),
    (dict(num_pages=1 << 31), {}, "num_pages"), (dict(reserved=1), {}, "reserved"), (dict(k_pool=None), {}, "NULL pool"),
    (dict(v_pool=8200), {}, "aligned"), ({}, dict(block_table=None), "NULL block_table"),
    ({}, dict(token_start=None), "NULL"), ({}, dict(ctx_lens=None), "NULL"), ({}, dict(n_seqs=0), "0 sequences"),
    ({}, dict(n_seqs=65536), "65536 sequences"), ({}, dict(table_stride=0), "table_stride 0"),
    ({}, dict(table_stride=1 << 25), "table_stride"), ({}, dict(n_tokens=1 << 23), "tokens"),
    ({}, dict(max_tokens=0), "max_tokens 0"), ({}, dict(reserved=1), "reserved"),
]
MASKED = ({}, dict(tree_mask=64, mask_words=0), "mask words")


@pytest.mark.parametrize("c,b,want", SHARED + [MASKED])
def test_cache_and_batch_are_checked_by_every_entry_point(c, b, want):
    lib = abi.load()
    st, msg = attn(cache(**c), batch(**b))
    assert st == abi.G4_EINVAL and want in msg, msg
    n = C.c_size_t(0)
    assert lib.g4_paged_attn_workspace_size(cache(**c), batch(**b), 8, C.byref(n)) == abi.G4_EINVAL
    p = abi.PagedAppendParams(8, 1e-6, 0, 0, 0)
    st = lib.g4_paged_append(cache(**c), batch(**b), 256, 256, 256, 256, 256, 256, 256, p, None)
    assert st == abi.G4_EINVAL and want in lib.g4_last_error().decode()
    if "tree_mask" in b:
        return  # the commit reads no masks
    st = lib.g4_paged_commit(cache(**c), 1, batch(**b), 64, 4, 64, 128, None)
    assert st == abi.G4_EINVAL and want in lib.g4_last_error().decode()


def test_attention_arguments():
    ok = (cache(), batch())
    for kw, want in [(dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict(ws=None), "NULL"), (dict(out=264), "aligned"),
                     (dict(q=258), "aligned"), (dict(ws=260), "aligned"), (dict(nqh=9), "9 query heads"),
                     (dict(nqh=0), "0 query heads"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                     (dict(cap=-1.0), "softcap"), (dict(cap=float("nan")), "softcap"), (dict(cap=1e-9), "softcap")]:
        st, msg = attn(*ok, **kw)
        assert st == abi.G4_EINVAL and want in msg, (kw, msg)
    assert attn(cache(num_kv_heads=3), batch(), nqh=8)[0] == abi.G4_EINVAL
    st, msg = attn(*ok, size=100)
    assert st == abi.G4_ENOSPC and "workspace" in msg
    assert attn(None, batch())[0] == abi.G4_EINVAL and attn(cache(), None)[0] == abi.G4_EINVAL
    assert attn(cache(), batch(n_tokens=0))[0] == abi.G4_OK  # nothing to do, nothing enqueued
    st, msg = attn(cache(num_kv_heads=64), batch(n_seqs=60000, n_tokens=1 << 22, max_tokens=1 << 20), nqh=512)
    assert st == abi.G4_EINVAL and "too much" in msg


def test_workspace_is_bounded_and_independent_of_the_lengths():
    lib = abi.load()
    sizes = []
    for b in (batch(), batch(table_stride=10000), batch(n_seqs=4000)):
        n = C.c_size_t(0)
        assert lib.g4_paged_attn_workspace_size(cache(), b, 8, C.byref(n)) == abi.G4_OK
        sizes.append(n.value)
    assert sizes[1] == sizes[0] and max(sizes) < 1 << 28


def test_append_arguments():
    lib = abi.load()

    def call(q=256, k=256, v=256, qw=256, kw=256, inv=256, qo=256, b=None, **p):
        d = dict(num_q_heads=8, eps=1e-6, q_stride=0, k_stride=0, v_stride=0)
        d.update(p)
        st = lib.g4_paged_append(cache(), batch(**(b or {})), q, k, v, qw, kw, inv, qo, abi.PagedAppendParams(**d), None)
        return st, lib.g4_last_error().decode()

    for kw, want in [(dict(inv=None), "rope_inv_freq"), (dict(q=None), "go together"), (dict(qo=None), "go together"),
                     (dict(v=None), "go together"), (dict(kw=None), "go together"), (dict(num_q_heads=0), "num_q_heads"),
                     (dict(q=None, qw=None, qo=None, k=None, v=None, kw=None), "neither"), (dict(eps=-1.0), "eps"),
                     (dict(eps=float("nan")), "eps"), (dict(q_stride=100), "stride"), (dict(k_stride=255), "stride"),
                     (dict(v_stride=1 << 40), "stride"), (dict(q_stride=2050), "aligned"), (dict(q=260), "aligned"),
                     (dict(qo=258), "aligned")]:
        st, msg = call(**kw)
        assert st == abi.G4_EINVAL and want in msg, (kw, msg)
    assert lib.g4_paged_append(cache(), batch(), 256, 256, 256, 256, 256, 256, 256, None, None) == abi.G4_EINVAL
    assert call(b=dict(n_tokens=0))[0] == abi.G4_OK


def test_commit_arguments():
    lib = abi.load()
    two = (abi.PagedCache * 65)(*[cache() for _ in range(65)])
    two[1].num_pages = 99

    def call(c=two, n=1, b=None, path=64, stride=4, acc=64, new=128):
        st = lib.g4_paged_commit(c, n, batch(**(b or {})), path, stride, acc, new, None)
        return st, lib.g4_last_error().decode()

    for kw, want in [(dict(n=0), "0 caches"), (dict(n=65), "65 caches"), (dict(n=2), "cache 1"), (dict(path=None), "NULL"),
                     (dict(acc=None), "NULL"), (dict(new=None), "NULL"), (dict(stride=0), "path_stride"),
                     (dict(new=64), "ctx_lens itself")]:
        st, msg = call(**kw)
        assert st == abi.G4_EINVAL and want in msg, (kw, msg)
    assert lib.g4_paged_commit(two, 1, None, 64, 4, 64, 128, None) == abi.G4_EINVAL


def test_logprobs_arguments():
    lib = abi.load()

    def call(logits=256, tokens=256, lp=256, ent=256, ids=256, tops=256, ws=256, size=1 << 40, **p):
        d = dict(rows=4, vocab=50000, row_stride=0, dtype=0, top_k=5, cap=0.0, temperature=1.0)
        d.update(p)
        p = abi.TokenLogprobsParams(**d)
        st = lib.g4_token_logprobs(logits, tokens, lp, ent, ids, tops, p, ws, size, None)
        return st, lib.g4_last_error().decode()

    for kw, want in [(dict(vocab=0), "vocab 0"), (dict(vocab=1 << 25), "vocab"), (dict(rows=65536), "rows"),
                     (dict(top_k=65), "top_k 65"), (dict(top_k=4, vocab=3), "top_k 4"), (dict(row_stride=100), "row_stride"),
                     (dict(dtype=3), "dtype 3"), (dict(cap=-1.0), "cap"), (dict(cap=float("nan")), "cap"),
                     (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                     (dict(temperature=float("nan")), "temperature"), (dict(logits=None), "NULL"), (dict(ws=None), "NULL"),
                     (dict(tokens=None), "go together"), (dict(lp=None), "go together"), (dict(ids=None), "top_ids"),
                     (dict(top_k=0), "top_ids"), (dict(logits=258), "misaligned"), (dict(ws=264), "aligned"),
                     (dict(tokens=None, lp=None, ent=None, ids=None, tops=None, top_k=0), "nothing")]:
        st, msg = call(**kw)
        assert st == abi.G4_EINVAL and want in msg, (kw, msg)
    st, msg = call(size=64)
    assert st == abi.G4_ENOSPC and "workspace" in msg
    assert call(rows=0)[0] == abi.G4_OK
    n = C.c_size_t(0)
    p = abi.TokenLogprobsParams(64, 262144, 0, 0, 20, 30.0, 1.0)
    assert lib.g4_token_logprobs_workspace_size(p, C.byref(n)) == abi.G4_OK and 0 < n.value < 1 << 20
    assert lib.g4_token_logprobs(256, 256, 256, None, None, None, None, 256, 1 << 30, None) == abi.G4_EINVAL


def test_tensor_wrappers_refuse_host_tensors_and_shapes():
    pool = torch.zeros(4, 16, 1, 256, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedCache(pool, pool)
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedBatch(torch.zeros(2, 4, dtype=torch.int32), pool, pool, 3)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_logprobs(torch.zeros(2, 8), None, None, None, None)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.token_logprobs(torch.zeros(8), None, None, None, None)


def test_commit_refuses_a_pool_twice_and_outputs_over_inputs():
    """Layers that share a cache name it once: two workgroups moving the same rows would each undo what the other
    relies on."""
    lib = abi.load()

    def call(caches, **kw):
        a = dict(b=batch(), path=0x10000, stride=4, acc=0x20000, new=0x30000)
        a.update(kw)
        c = (abi.PagedCache * len(caches))(*caches)
        st = lib.g4_paged_commit(c, len(caches), a["b"], a["path"], a["stride"], a["acc"], a["new"], None)
        return st, lib.g4_last_error().decode()

    apart = [cache(k_pool=0x1000000 * (2 * i + 1), v_pool=0x1000000 * (2 * i + 2)) for i in range(64)]
    for n, i, j in [(2, 0, 1), (17, 3, 16), (64, 0, 63), (64, 62, 63)]:
        for what in ("k_pool", "v_pool"):
            cs = [abi.PagedCache.from_buffer_copy(c) for c in apart[:n]]
            setattr(cs[j], what, getattr(cs[i], what))
            st, msg = call(cs)
            assert st == abi.G4_EINVAL and "twice" in msg, (n, i, j, what, msg)
    one = abi.PagedCache.from_buffer_copy(apart[0])
    one.v_pool = one.k_pool
    assert "twice" in call([one])[1]
    n = batch().n_seqs
    for kw in [dict(new=0x20000), dict(new=0x10000 + 4 * (4 * n - 1)), dict(new=0x20000 - 4 * (n - 1)),
               dict(acc=0x30000 + 4 * (n - 1)), dict(path=0x30000)]:
        st, msg = call(apart[:1], **kw)
        assert st == abi.G4_EINVAL and "lies over" in msg, (kw, msg)


@pytest.mark.parametrize("vocab", [1000, 50257, 131072, 131073, 151936, 262144, 1 << 20])
@pytest.mark.parametrize("k", [0, 5, 20, 64])
def test_a_workspace_serves_every_smaller_call(vocab, k):
    """A step with fewer rows, a smaller vocabulary or fewer alternatives than the workspace was sized for is not
    refused: the size never falls as one of them grows, over the row counts at which the chunks' length changes. (What
    a call needs is at most its own size.)"""
    lib = abi.load()

    def size(rows, v=vocab, top=k):
        n = C.c_size_t(0)
        assert lib.g4_token_logprobs_workspace_size(abi.TokenLogprobsParams(rows, v, 0, 0, top, 0.0, 1.0), C.byref(n)) == 0
        return n.value

    sizes = [size(r) for r in range(1, 600)] + [size(65535)]
    assert sizes == sorted(sizes)
    for r in (1, 3, 15, 16, 73, 74, 300, 600):
        by_vocab = [size(r, v) for v in sorted({1000, vocab // 2, vocab - 1, vocab, vocab + 1, 2 * vocab, 65536, 131072, 131073})]
        assert by_vocab == sorted(by_vocab), r
        assert size(r, top=k // 2) <= size(r)


def test_commit_refuses_new_lengths_over_what_other_workgroups_read():
    """One workgroup writes the lengths while others still look their sequence and their pages up."""
    lib = abi.load()
    b = batch(token_start=0x40000, block_table=0x50000, ctx_lens=0x60000)
    for new in (0x40000, 0x40000 + 4 * b.n_seqs, 0x40000 - 4 * (b.n_seqs - 1), 0x50000,
                0x50000 + 4 * (b.n_seqs * b.table_stride - 1), 0x50000 - 4 * (b.n_seqs - 1)):
        st = lib.g4_paged_commit(cache(k_pool=0x1000000, v_pool=0x2000000), 1, b, 0x10000, 4, 0x20000, new, None)
        assert st == abi.G4_EINVAL and "lies over" in lib.g4_last_error().decode(), hex(new)
