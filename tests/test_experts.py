"""The expert layer's operators without a GPU: descriptors, workspaces and refusals of the C ABI, and
arguments that are no device tensors."""
import ctypes
import os
import subprocess

import pytest
import torch

from mintccl_amd import _lib
from mintccl_amd.block8 import Blocks, product, quantise, quantise_weight, weight_grad
from mintccl_amd.combine import combine, combine_grad
from mintccl_amd.routing import Assignment, assign, route, route_grad

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mintccl.h")


@pytest.mark.parametrize("struct,name", [(_lib.RouteOp, "mint_route_op"), (_lib.ProductOp, "mint_product_op"),
                                         (_lib.WeightGradOp, "mint_weight_grad_op")])
def test_descriptor_layouts_match_the_header(tmp_path, struct, name):
    fields = [f for f, _ in struct._fields_]
    src = tmp_path / "layout.c"
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){", f'  printf("%zu\\n", sizeof({name}));']
    lines += [f'  printf("%zu\\n", offsetof({name}, {f}));' for f in fields]
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c11", "-o", str(exe), str(src)])
    out = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert out == [ctypes.sizeof(struct)] + [getattr(struct, f).offset for f in fields]


def make(struct, **kw):
    d = struct()
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def route_op(**kw):
    base = dict(logits=4096, weights=8192, chosen=12288, row_stride=64, tokens=5, experts=64, topk=6, groups=1, kept=1,
                group_top=1, dtype=_lib.F32, scale=1.0)
    return make(_lib.RouteOp, **{**base, **kw})


@pytest.mark.parametrize("code,kw", [
    (_lib.ERR_ARG, {"experts": 0}), (_lib.ERR_ARG, {"experts": 1025}), (_lib.ERR_ARG, {"topk": 0}), (_lib.ERR_ARG, {"topk": 65}),
    (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"score": 2}), (_lib.ERR_ARG, {"logits": 0}), (_lib.ERR_ARG, {"weights": 0}),
    (_lib.ERR_ARG, {"chosen": 0}), (_lib.ERR_ARG, {"tokens": 1 << 31}), (_lib.ERR_GEOMETRY, {"groups": 7}), (_lib.ERR_GEOMETRY, {"groups": 0}),
    (_lib.ERR_GEOMETRY, {"groups": 8, "kept": 9}), (_lib.ERR_GEOMETRY, {"group_top": 3}), (_lib.OK, {"tokens": 0, "logits": 0})])
def test_route_refuses(code, kw):
    assert _lib.lib().mint_route(route_op(**kw), None) == code


def test_route_grad_and_assign_refuse():
    L = _lib.lib()
    assert L.mint_route(None, None) == L.mint_route_grad(None, 0, 0, 0, None) == _lib.ERR_ARG
    assert L.mint_route_grad(route_op(), 0, 4096, 64, None) == _lib.ERR_ARG
    assert L.mint_route_grad(route_op(tokens=0), 0, 0, 64, None) == _lib.OK
    assign_ = lambda chosen=4096, t=5, k=2, first=0, n=8, off=4096, order=4096, slots=4096, room=None, size=0: L.mint_assign(  # noqa: E731
        chosen, t, k, first, n, off, order, slots, room, size, None)
    assert assign_(n=0) == assign_(n=1025) == assign_(k=0) == assign_(off=None) == assign_(chosen=None) == _lib.ERR_ARG
    assert assign_(first=2 ** 31 - 4) == _lib.ERR_ARG
    assert assign_(t=2 ** 31) == _lib.ERR_TOO_LARGE
    need = L.mint_assign_workspace(100000 * 2, 8)
    assert need > 0 and L.mint_assign_workspace(4096, 8) == 0
    assert assign_(t=100000) == assign_(t=100000, room=4096, size=need - 1) == _lib.ERR_STAGING


def product_op(**kw):
    base = dict(kind=0, dtype=_lib.BF16, x=4096, w=4096, sx=4096, sw=4096, out=4096, rows=4, cols=8, depth=256, x_rows=4, x_stride=256,
                w_stride=256, out_stride=8, sx_row=2, sx_block=1, sw_row=2, sw_block=1, x_dtype=_lib.BYTES)
    return make(_lib.ProductOp, **{**base, **kw})


@pytest.mark.parametrize("code,kw", [
    (_lib.ERR_ARG, {"kind": 2}), (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"x_dtype": 7}), (_lib.ERR_ARG, {"out": 0}),
    (_lib.ERR_ARG, {"x": 0}), (_lib.ERR_ARG, {"w": 0}), (_lib.ERR_ARG, {"sx": 0}), (_lib.ERR_ARG, {"sw": 0}), (_lib.ERR_ARG, {"x_rows": 3}),
    (_lib.ERR_ARG, {"experts": 2}), (_lib.ERR_ARG, {"kind": 1, "x_dtype": _lib.F32}), (_lib.ERR_ALIGN, {"x": 4104}),
    (_lib.ERR_ALIGN, {"w": 4104}), (_lib.ERR_ALIGN, {"x_stride": 250}), (_lib.ERR_ALIGN, {"w_stride": 250}),
    (_lib.ERR_ALIGN, {"w_matrix": 8}), (_lib.ERR_GEOMETRY, {"kind": 1, "depth": 200}), (_lib.ERR_TOO_LARGE, {"rows": 1 << 31, "x_rows": 1 << 31}),
    (_lib.ERR_STAGING, {"x_dtype": _lib.F32, "rows": 400, "x_rows": 400}), (_lib.OK, {"rows": 0, "out": 0}), (_lib.OK, {"cols": 0, "out": 0})])
def test_product_refuses(code, kw):
    assert _lib.lib().mint_product8(product_op(**kw), None) == code


def test_workspaces():
    L = _lib.lib()
    room = lambda **kw: L.mint_product8_workspace(product_op(**kw))  # noqa: E731
    assert room() == 0                                              # in 8 bits already
    assert room(x_dtype=_lib.F32) == 0                              # few rows: rounded on the way
    assert room(x_dtype=_lib.F32, rows=400, x_rows=400) == 400 * 2 * 132
    grad = make(_lib.WeightGradOp, rows=300, x_rows=300, cols=10, depth=20)
    assert L.mint_weight_grad8_workspace(grad) == 3 * 128 * 30 + 3 * 30 * 4
    grad.experts = 5
    assert L.mint_weight_grad8_workspace(grad) == 8 * 128 * 30 + 8 * 30 * 4
    assert L.mint_columns8_blocks(300, 5) == 8


def test_workspace_of_a_shared_tile():
    """Few tiles of 64 x 64 and a long depth: sums of four wavefronts, 16 KiB a tile and part, and their counts, behind what is rounded."""
    L = _lib.lib()
    op = product_op(rows=64, x_rows=64, cols=4096, depth=4096)
    sums = 64 * 4 * 16384 + 64 * 4 * 4
    assert L.mint_product8_workspace(op) == sums
    op.x_dtype = _lib.F32
    assert L.mint_product8_workspace(op) == 64 * 32 * 132 + sums
    op.depth = 31 * 128                                      # (results in 16 bits: not worth it)
    assert L.mint_product8_workspace(op) == 64 * 31 * 132



def test_weight_grad_rounding_and_combination_refuse():
    L = _lib.lib()
    base = dict(d=4096, x=4096, out=4096, rows=300, x_rows=300, cols=10, depth=20, d_dtype=2, x_dtype=2, dtype=2)
    go = lambda **kw: L.mint_weight_grad8(make(_lib.WeightGradOp, **{**base, **kw}), None)  # noqa: E731
    assert go() == _lib.ERR_STAGING
    assert go(d=0) == go(x=0) == go(out=0) == go(dtype=3) == go(experts=2) == go(x_rows=200) == _lib.ERR_ARG
    assert go(rows=1 << 31) == _lib.ERR_TOO_LARGE and go(cols=0) == _lib.OK
    rows8 = lambda x=4096, rows=4, depth=200, dt=2, q=4096, stride=256, s=4096: L.mint_rows8(x, 200, rows, depth, dt, q, stride, s, 1, 4, None)  # noqa: E731
    assert rows8(dt=3) == rows8(x=None) == rows8(s=None) == _lib.ERR_ARG
    assert rows8(q=4104) == rows8(stride=264) == _lib.ERR_ALIGN and rows8(stride=128) == _lib.ERR_GEOMETRY and rows8(rows=0) == _lib.OK
    cols8 = lambda x=4096, n=4, stride=128, tokens=None, off=None, e=0, rows=4: L.mint_columns8(x, 8, n, 8, 2, tokens, rows, off, e, 4096, stride, 4096, None)  # noqa: E731
    assert cols8(x=None) == cols8(n=3) == cols8(e=2) == cols8(n=0, tokens=4096) == _lib.ERR_ARG
    assert cols8(stride=112) == _lib.ERR_GEOMETRY and cols8(rows=0) == _lib.OK
    squares = lambda w=4096, n=1, stride=256, q=4096: L.mint_squares8(w, 0, 200, n, 8, 200, 2, q, 2048, stride, 4096, None)  # noqa: E731
    assert squares(w=None) == _lib.ERR_ARG and squares(q=4100) == _lib.ERR_ALIGN and squares(stride=128) == _lib.ERR_GEOMETRY
    assert squares(n=0) == _lib.OK and squares(n=70000) == _lib.ERR_TOO_LARGE
    comb = lambda rows=4096, slots=4096, t=4, k=2, out=4096, dt=2, width=8: L.mint_combine(rows, 8, 8, slots, None, t, k, width, out, 8, dt, None)  # noqa: E731
    assert comb(rows=None) == comb(slots=None) == comb(out=None) == comb(k=0) == comb(dt=3) == _lib.ERR_ARG
    assert comb(t=1 << 31) == _lib.ERR_TOO_LARGE and comb(t=0) == comb(width=0) == _lib.OK
    back = lambda d=4096, used=4096, t=4, n=8, d_rows=4096: L.mint_combine_grad(d, 8, 4096, 8, n, 4096, None, used, t, 2, 8, d_rows, 8, None, 2, None)  # noqa: E731
    assert back(d=None) == back(used=None) == back(d_rows=None) == _lib.ERR_ARG and back(t=0, n=0) == _lib.OK
    assert back(t=1 << 30) == _lib.ERR_TOO_LARGE


def test_the_operators_take_device_tensors():
    x, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    plan, w = Assignment(i[0], i[0], i), Blocks(x, x)
    for call in (lambda: route(x, 2), lambda: route_grad(x, x, i), lambda: assign(i, 4), lambda: quantise(x), lambda: quantise_weight(x),
                 lambda: product(x, w), lambda: weight_grad(x, x), lambda: combine(x, plan), lambda: combine_grad(x, x, plan),
                 lambda: quantise(None), lambda: combine(3, plan)):
        with pytest.raises(TypeError, match="device tensor"):
            call()
    with pytest.raises(ValueError, match="score"):
        route(x, 2, score="tanh")
    with pytest.raises(TypeError, match="float16, bfloat16"):
        product(x, w, dtype=torch.int8)


def test_the_gradients_product_refuses_fewer_rows_than_its_result():
    assert _lib.lib().mint_product8(product_op(kind=1, rows=5, x_rows=4, sw_row=1), None) == _lib.ERR_ARG
