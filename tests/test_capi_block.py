"""CPU-side checks of the C ABI around an expert block: the descriptors' layout, and the argument errors that come before a GPU is touched."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "fast_moe_amd.h")
ANY = 1 << 20       # (an address that is never followed)


@pytest.fixture(scope="module")
def lib():
    from fast_moe_amd.kernels.hip import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from fast_moe_amd import build
        build.build(verbose=False)
    return _lib.load()


def refuses(lib, call, code, message):
    assert call() == code
    assert re.search(message, lib.fmoe_last_error().decode()), lib.fmoe_last_error()


@pytest.mark.parametrize("struct,cls", [("fmoe_few_desc", "FewDesc"), ("fmoe_norm_desc", "NormDesc")])
def test_descriptors_are_the_headers(struct, cls, tmp_path):
    from fast_moe_amd.kernels.hip import _lib
    desc = getattr(_lib, cls)
    names = [f[0] for f in desc._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {", f'  printf("%zu\\n", sizeof({struct}));']
    prog += [f'  printf("%zu\\n", offsetof({struct}, {n}));' for n in names] + ["  return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(prog))
    subprocess.run(["gcc", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")], check=True)
    out = [int(v) for v in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(desc) and out[1:] == [getattr(desc, n).offset for n in names]
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), text, flags=re.S).group(1)
    assert [n for stmt in body.split(";") if stmt.strip() for n in re.findall(r"(\w+)\s*(?:,|$)", stmt.strip())] == names


def test_enumerators_are_the_headers():
    from fast_moe_amd.kernels.hip import _lib
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    enums = {n: int(v) for n, v in re.findall(r"\b(FMOE_[A-Z0-9_]+)\s*=\s*(-?\d+)", text)}
    assert (enums["FMOE_NORM_RMS"], enums["FMOE_NORM_LAYER"]) == (_lib.NORM_RMS, _lib.NORM_LAYER)
    assert (enums["FMOE_GATE_TOKEN"], enums["FMOE_GATE_ELEMENT"]) == (_lib.ROW_GATE_TOKEN, _lib.ROW_GATE_ELEMENT)


def few(**kw):
    from fast_moe_amd.kernels.hip import _lib
    d = _lib.FewDesc()
    d.T, d.E, d.k, d.D, d.H, d.O, d.dtype, d.weight_dtype = 4, 8, 2, 64, 32, 64, _lib.FMOE_BF16, _lib.FMOE_BF16
    for n in ("x", "gate_weight", "w", "wo", "out"):
        setattr(d, n, ANY)
    d.x_stride_row, d.gate_stride_row, d.w_stride_e, d.w_stride_n, d.wo_stride_e, d.wo_stride_n, d.out_stride_row = 64, 64, 64 * 32, 64, 64 * 32, 32, 64
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def test_few_tokens_refuses_without_a_gpu(lib):
    from fast_moe_amd.kernels.hip import _lib
    run = lambda d, ws=ANY, n=1 << 30: lib.fmoe_few_tokens(ctypes.byref(d) if d is not None else None, ws, n, None)
    refuses(lib, lambda: run(None), 1, "desc is NULL")
    for bad, message in ((dict(T=65), "up to 64 tokens"), (dict(T=-1), "up to 64 tokens"), (dict(E=257), "E <= 256"), (dict(k=17, E=32), "k <= 16"), (dict(k=9), "k <= E"),
                         (dict(k=0), "1 <= k"), (dict(D=0), "widths"), (dict(H=65537), "widths"), (dict(dtype=_lib.FMOE_E4M3), "tokens must be"),
                         (dict(weight_dtype=_lib.FMOE_F32), "weights must have"), (dict(dtype=_lib.FMOE_F32, weight_dtype=_lib.FMOE_E4M3), "weights must have"),
                         (dict(weight_dtype=_lib.FMOE_E4M3), "need their scales"), (dict(wo=None), "NULL tensor"), (dict(bias_p=ANY), "goes with wp"),
                         (dict(x_stride_row=63), "rows overlap"), (dict(w_stride_n=63), "rows overlap"), (dict(w_stride_e=-1), "rows overlap"),
                         (dict(out_stride_row=63), "rows overlap"), (dict(wo_stride_n=(1 << 20) + 1), "row strides")):
        d = few(**bad)
        refuses(lib, lambda: run(d), 1, message)
        assert lib.fmoe_few_tokens_workspace_bytes(ctypes.byref(d)) == 0
    need = lib.fmoe_few_tokens_workspace_bytes(ctypes.byref(few()))
    assert need > 4 * 2 * 32 * 2
    refuses(lib, lambda: run(few(), ANY, need - 1), 3, "workspace")
    refuses(lib, lambda: run(few(), None, need), 3, "workspace")
    refuses(lib, lambda: run(few(), ANY + 8, need), 1, "16-byte aligned")
    assert run(few(T=0, x=None), None, 0) == 0              # nothing to do


def norm(**kw):
    from fast_moe_amd.kernels.hip import _lib
    d = _lib.NormDesc()
    d.rows, d.cols, d.dtype, d.param_dtype = 4, 64, _lib.FMOE_BF16, _lib.FMOE_F32
    for n in ("y", "residual", "weight", "next_weight", "out", "next"):
        setattr(d, n, ANY)
    d.y_stride = d.residual_stride = 64
    for n, v in kw.items():
        setattr(d, n, v)
    return d


def test_norms_refuse_without_a_gpu(lib):
    from fast_moe_amd.kernels.hip import _lib
    forward = lambda d: lib.fmoe_norm_add(ctypes.byref(d), None)
    for bad, message in ((dict(rows=-1), "rows >= 0"), (dict(cols=0), "1 to 8192"), (dict(cols=8193), "1 to 8192"), (dict(dtype=_lib.FMOE_E4M3), "bf16 or fp32"),
                         (dict(param_dtype=7), "parameters"), (dict(norm=2), "unknown norm"), (dict(gate_mode=3), "unknown gate"), (dict(gate_mode=1), "a gate needs"),
                         (dict(weight=None, bias=ANY), "goes with weight"), (dict(next_weight=None, next_bias=ANY), "goes with next_weight"),
                         (dict(residual=None), "residual"), (dict(next_weight=None), "nothing to write"), (dict(y=None), "out without y"),
                         (dict(K=2, value_rows=8), "a merge needs"), (dict(K=2, reverse_index=ANY, value_rows=7), "a merge needs"),
                         (dict(K=65, reverse_index=ANY, value_rows=260), "K <= 64"), (dict(stats=ANY + 8), "16-byte aligned")):
        d = norm(**bad)
        refuses(lib, lambda: forward(d), 1, message)
    refuses(lib, lambda: lib.fmoe_norm_add(None, None), 1, "desc is NULL")
    assert forward(norm(rows=0, residual=None)) == 0
    given = dict(stats=ANY, d_out=ANY, d_y=ANY)
    backward = lambda d: lib.fmoe_norm_add_bwd(ctypes.byref(d), None, 0, None)
    for bad, message in ((dict(stats=None), "stats and a gradient"), (dict(d_out=None), "stats and a gradient"), (dict(K=1, value_rows=4), "merged rows"), (dict(d_merge=ANY), "not there"),
                         (dict(next_weight=None, d_next=ANY), "d_next needs"), (dict(d_scale=ANY), "not there"), (dict(d_gate=ANY), "not there"),
                         (dict(d_bias=ANY), "not there"), (dict(y=None), "not there")):
        d = norm(**dict(given, **bad))
        refuses(lib, lambda: backward(d), 1, message)
        assert lib.fmoe_norm_add_bwd_workspace_bytes(ctypes.byref(d)) == 0
    d = norm(**dict(given, d_weight=ANY))
    assert lib.fmoe_norm_add_bwd_workspace_bytes(ctypes.byref(d)) >= 64 * 4
    refuses(lib, lambda: backward(d), 3, "workspace")


def test_checkpoints_refuse_without_a_gpu(lib):
    assert [lib.fmoe_swiglu_checkpoint_cols(n) for n in (1, 32, 33, 1408)] == [32, 32, 64, 1408]
    write = lambda g=ANY, dtype=1, rows=4, cols=64, gs=64, us=64, q=ANY: lib.fmoe_swiglu_checkpoint(g, ANY, dtype, rows, cols, gs, us, q, ANY, None)
    for bad, message in ((dict(dtype=5), "bf16 or fp32"), (dict(rows=-1), "rows >= 0"), (dict(cols=0), "columns"), (dict(q=None), "NULL"), (dict(q=ANY + 8), "aligned"),
                         (dict(g=None), "NULL"), (dict(us=63), "overlap"), (dict(rows=1 << 40, cols=1 << 24, gs=1 << 24, us=1 << 24), "too many")):
        refuses(lib, lambda: write(**bad), 1, message)
    assert write(rows=0, g=None, q=None) == 0
    back = lambda d=ANY, wt=0, ds=64, dgs=64, hs=64, w=ANY: lib.fmoe_swiglu_checkpoint_bwd(ANY, ANY, d, 1, 4, 64, ds, w, wt, ANY, ANY, dgs, ANY, hs, None, None)
    for bad, message in ((dict(d=None), "NULL"), (dict(wt=9), "row weights"), (dict(ds=63), "overlap"), (dict(dgs=63), "overlap"), (dict(hs=63), "overlap")):
        refuses(lib, lambda: back(**bad), 1, message)
