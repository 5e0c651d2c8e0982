"""Operands of the operators between two attention blocks that share memory, on the CPU: the predicate against marked bytes, and
the calls whose outputs lie over rows that they or other workgroups still read, refused before anything is enqueued. Calls that
may share memory stay what they were: they are made with no tokens, or by the GPU tests."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from g4attn import abi

HERE = Path(__file__).resolve().parent


def test_the_predicate(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ is not installed")
    exe = tmp_path / "row_ranges_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    str(HERE / "row_ranges_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, (out.returncode, out.stdout)


def refused(status, want):
    msg = abi.load().g4_last_error().decode()
    assert status == abi.G4_EINVAL and want in msg, (status, msg)


# Operands far apart: 64 elements a row, 16 rows.
X, RES, POST, W, SUM, OUT, SCALES, IDS, A, B, SPACE, BASE = ((i + 1) << 24 for i in range(12))


def norm(x=X, residual=RES, post=POST, weight=W, total=SUM, out=OUT, scales=None, **kw):
    p = dict(rows=16, n=64, x_type=0, residual_type=0, weight_type=1, out_type=0, eps=1e-6, reserved=0, x_stride=0,
             residual_stride=0, residual_out_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_add_rms_norm(x, residual, post, weight, total, out, scales, abi.AddRmsNormParams(**p), None)


@pytest.mark.parametrize("args,want", [
    # a view shifted by a row, by an element, and one that begins before
    (dict(out=X + 256), "out lies over x"), (dict(out=X + 4), "out lies over x"), (dict(out=X - 256 * 15), "out lies over x"),
    (dict(out=RES + 256), "out lies over residual"), (dict(total=X + 256), "residual_out lies over x"),
    (dict(total=RES - 256), "residual_out lies over residual"), (dict(out=X + 2048, out_type=1), "out lies over x"),
    (dict(out=X + 512, out_type=3, scales=SCALES), "out lies over x"),
    # rows beside others, by an element too far
    (dict(x_stride=128, out=X + 252, out_stride=128), "out lies over x"), (dict(x_stride=128, out=X + 260, out_stride=128), "out lies over x"),
    (dict(out=SUM + 256), "out lies over residual_out"), (dict(out=W - 512), "out lies over weight"), (dict(total=POST), "over post_weight"),
    (dict(out=W - 4096 + 4), "out lies over weight"), (dict(total=W + 124), "residual_out lies over weight"),
    (dict(out_type=3, scales=X + 1024), "scales lies over x"), (dict(out_type=3, scales=RES), "scales lies over residual"),
    (dict(out_type=3, scales=W), "scales lies over weight"), (dict(out_type=3, scales=OUT + 1020), "out lies over scales"),
    (dict(out_type=3, scales=SUM), "residual_out lies over scales"),
])
def test_add_rms_norm(args, want):
    refused(norm(**args), want)


@pytest.mark.parametrize("x,out,scales,kw,want", [
    (X, X + 256, SCALES, {}, "out lies over x"), (X, X - 64, SCALES, {}, "out lies over x"), (X, OUT, X + 4, {}, "scales lies over x"),
    (X, OUT, OUT + 64, {}, "out lies over scales"), (X, X + 64, SCALES, dict(x_stride=80, out_stride=320), "out lies over x"),
])
def test_quantize_rows(x, out, scales, kw, want):
    p = dict(rows=16, n=64, x_type=0, reserved=0, x_stride=0, out_stride=0)
    p.update(kw)
    refused(abi.load().g4_quantize_rows(x, out, scales, abi.QuantizeRowsParams(**p), None), want)


def lora():
    return abi.Lora(a=A, b=B, scales=SCALES, n_adapters=4, rank=16, n=64, n_segs=2, widths=(C.c_uint32 * 4)(40, 24, 0, 0), type=1,
                    reserved=0)


def lora_add(ids=IDS, x=X, xs=None, base=BASE, out=OUT, space=SPACE, **kw):
    p = dict(n_tokens=16, x_type=1, out_type=0, reserved=0, x_stride=0, base_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_lora_add(lora(), ids, x, xs, base, out, abi.LoraAddParams(**p), space, 1 << 20, None)


@pytest.mark.parametrize("args,want", [
    (dict(out=BASE + 256), "out lies over base"), (dict(out=BASE - 4), "out lies over base"),
    (dict(base_stride=128, out=BASE + 252, out_stride=128), "out lies over base"),
    (dict(out=B + 512), "out lies over the adapters' up rows"), (dict(out=SCALES), "out lies over the adapters' scales"),
    (dict(out=IDS - 512), "out lies over adapter_ids"), (dict(space=X), "workspace lies over x"), (dict(space=A + 64), "over the adapters' down rows"),
    (dict(space=BASE), "workspace lies over base"), (dict(out=SPACE + 64), "workspace lies over out"), (dict(ids=SPACE), "workspace lies over adapter_ids"),
    (dict(x_type=3, xs=SPACE + 64), "workspace lies over x_scales"),
])
def test_lora_add(args, want):
    refused(lora_add(**args), want)


def linear(low=None, ids=None, x=X, xs=RES, w=W, ws=POST, out=OUT, space=SPACE, **kw):
    p = dict(n_tokens=16, rows=64, n=64, out_type=0, x_stride=0, out_stride=0)
    p.update(kw)
    return abi.load().g4_linear_e4m3(x, xs, w, ws, low, ids, out, abi.LinearE4m3Params(**p), space, 1 << 20, None)


@pytest.mark.parametrize("args,want", [
    (dict(out=X), "out lies over x"), (dict(out=X - 4096 + 4), "out lies over x"), (dict(out=W + 128), "out lies over weight"),
    (dict(out=RES), "out lies over x_scales"), (dict(out=POST - 64), "out lies over weight_scales"),
    (dict(x_stride=320, out=X + 60, out_stride=80), "out lies over x"),
    (dict(low=True, out=SPACE), "workspace lies over out"), (dict(low=True, out=B), "out lies over the adapters' up rows"),
    (dict(low=True, out=IDS), "out lies over adapter_ids"), (dict(low=True, space=W), "workspace lies over weight"),
    (dict(low=True, space=X), "workspace lies over x"),
])
def test_linear_e4m3(args, want):
    args = dict(args)
    if args.pop("low", False):
        args.update(low=lora(), ids=IDS)
    refused(linear(**args), want)
