"""The operators around an expert layer without a GPU: descriptors, workspaces and refusals of the C ABI, arguments that are no device
tensors, and the oracle's gradients against differences."""
import ctypes
import os
import subprocess

import pytest
import torch

from mintccl_amd import _lib
from mintccl_amd.dense import activation_grad, input_grad, product, weight_grad
from mintccl_amd.norms import Norm, join, join_grad, norm, norm_grad
from mintccl_amd.routing import Balance, balance, balance_grad
from tests.block_oracle import activated64, balance64, gate64, join_grad64, norm64, norm_grad64, slope64

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mintccl.h")


@pytest.mark.parametrize("struct,name", [(_lib.NormSpec, "mint_norm"), (_lib.JoinOp, "mint_join_op"), (_lib.JoinGradOp, "mint_join_grad_op"),
                                         (_lib.DenseOp, "mint_dense_op"), (_lib.ActivationGradOp, "mint_activation_grad_op"),
                                         (_lib.BalanceOp, "mint_balance_op")])
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


def spec(**kw):
    return make(_lib.NormSpec, **{**dict(weight=4096, kind=1, dtype=_lib.BF16, eps=1e-5), **kw})


def join_op(**kw):
    base = dict(stream=4096, y=8192, new_stream=12288, next=16384, stream_stride=64, y_stride=64, new_stride=64, next_stride=64, rows=5, width=64,
                before=spec(), stream_dtype=_lib.F32, dtype=_lib.BF16, scale=1.0, carry=1.0)
    return make(_lib.JoinOp, **{**base, **kw})


BAD_JOINS = [
    (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"stream_dtype": _lib.F16}), (_lib.ERR_ARG, {"stream": 0}), (_lib.ERR_ARG, {"new_stream": 0}),
    (_lib.ERR_ARG, {"gate_by": 1, "gate": 4096, "gate_form": 1}), (_lib.ERR_ARG, {"gate": 4096, "gate_form": 0}), (_lib.ERR_ARG, {"gate": 4096, "gate_form": 4}),
    (_lib.ERR_ARG, {"gate": 4096, "gate_form": 1, "gate_dtype": _lib.BYTES}), (_lib.ERR_ARG, {"before": spec(kind=0)}), (_lib.ERR_ARG, {"before": spec(kind=3)}),
    (_lib.ERR_ARG, {"before": spec(dtype=3)}), (_lib.ERR_ARG, {"after": spec(kind=-1)}), (_lib.ERR_ARG, {"y": 0, "after": spec()}),
    (_lib.ERR_ARG, {"y": 0, "next": 0}), (_lib.ERR_ARG, {"y": 0, "gate": 4096, "gate_form": 1}), (_lib.ERR_TOO_LARGE, {"rows": 1 << 30}),
    (_lib.ERR_TOO_LARGE, {"width": 1 << 31}), (_lib.ERR_TOO_LARGE, {"rows": 1 << 27, "width": 20000}), (_lib.OK, {"rows": 0, "stream": 0}), (_lib.OK, {"width": 0})]


@pytest.mark.parametrize("code,kw", BAD_JOINS)
def test_join_refuses(code, kw):
    assert _lib.lib().mint_join(join_op(**kw), None) == code


@pytest.mark.parametrize("code,kw,of_join", [
    (_lib.ERR_ARG, {}, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"d_stream": 0, "d_next": 0}, {}), (_lib.ERR_ARG, {}, {"stream": 0}),
    (_lib.ERR_ARG, {}, {"before": spec(kind=0, weight=0)}), (_lib.ERR_ARG, {"to_gate": 4096}, {}), (_lib.ERR_ARG, {"to_before_bias": 4096}, {}),
    (_lib.ERR_ARG, {"to_after_weight": 4096}, {}), (_lib.ERR_ARG, {"to_y": 4096}, {"y": 0}), (_lib.ERR_STAGING, {"workspace": 0}, {}),
    (_lib.ERR_STAGING, {"workspace_bytes": 4}, {}), (_lib.ERR_ALIGN, {"workspace": 4098}, {}), (_lib.OK, {}, {"width": 0}),
    (_lib.OK, {"to_before_weight": 0, "workspace": 0}, {"rows": 0, "stream": 0, "y": 0})])
def test_join_grad_refuses(code, kw, of_join):
    base = dict(join=join_op(**of_join), d_stream=4096, d_next=8192, to_stream=12288, to_y=16384 if of_join.get("y", 1) else 0, to_before_weight=20480,
                workspace=1 << 20, workspace_bytes=1 << 20)
    assert _lib.lib().mint_join_grad(make(_lib.JoinGradOp, **{**base, **kw}), None) == code


def test_join_grad_workspace():
    L = _lib.lib()
    room = lambda **kw: L.mint_join_grad_workspace(make(_lib.JoinGradOp, **{**dict(join=join_op(), to_before_weight=4096), **kw}))  # noqa: E731
    # (four narrow rows a thread block, a line of sums for each of its vectors)
    assert room() == 2 * 2 * 64 * 4 and room(to_before_weight=0) == 0 and room(join=join_op(y=0)) == 2 * 64 * 4
    assert room(join=join_op(rows=0)) == 0 and room(join=join_op(before=spec(bias=4096))) == 2 * 4 * 64 * 4
    gated = join_op(gate=4096, gate_form=1, gate_dtype=_lib.F32)
    assert room(join=gated, to_before_weight=0, to_gate=4096) > 0 and room(join=join_op(gate=4096, gate_form=3), to_before_weight=0, to_gate=4096) == 0
    assert L.mint_join_grad_workspace(None) == 0 and L.mint_join(None, None) == L.mint_join_grad(None, None) == _lib.ERR_ARG


def dense_op(**kw):
    base = dict(form=0, dtype=_lib.BF16, out_dtype=_lib.BF16, x=4096, w=8192, out=12288, rows=5, cols=64, depth=64, x_stride=64, w_stride=64, out_stride=64)
    return make(_lib.DenseOp, **{**base, **kw})


@pytest.mark.parametrize("code,kw", [
    (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"out_dtype": _lib.F16}), (_lib.ERR_ARG, {"form": 3}), (_lib.ERR_ARG, {"form": -1}),
    (_lib.ERR_ARG, {"activation": 7}), (_lib.ERR_ARG, {"activation": -1}), (_lib.ERR_ARG, {"x": 0}), (_lib.ERR_ARG, {"w": 0}), (_lib.ERR_ARG, {"out": 0}),
    (_lib.ERR_ARG, {"form": 1, "bias": 4096}), (_lib.ERR_ARG, {"form": 1, "activation": 2}), (_lib.ERR_ARG, {"form": 2, "residual": 4096}), (_lib.ERR_ARG, {"form": 2, "z": 4096}),
    (_lib.ERR_TOO_LARGE, {"rows": 1 << 31}), (_lib.ERR_TOO_LARGE, {"cols": 1 << 31}), (_lib.ERR_TOO_LARGE, {"depth": 1 << 31}),
    (_lib.ERR_STAGING, {"rows": 64, "depth": 65536}), (_lib.ERR_STAGING, {"rows": 64, "depth": 65536, "workspace": 4096, "workspace_bytes": 64}),
    (_lib.ERR_ALIGN, {"rows": 64, "depth": 65536, "workspace": 4104, "workspace_bytes": 1 << 30}), (_lib.OK, {"rows": 0, "x": 0}), (_lib.OK, {"cols": 0, "w": 0})])
def test_dense_refuses(code, kw):
    assert _lib.lib().mint_dense(dense_op(**kw), None) == code


def test_dense_workspace():
    L = _lib.lib()
    assert L.mint_dense_workspace(None) == 0 and L.mint_dense(None, None) == _lib.ERR_ARG and L.mint_activation_grad(None, None) == _lib.ERR_ARG
    assert L.mint_dense_workspace(dense_op(rows=1)) == 0 and L.mint_dense_workspace(dense_op(rows=8192, cols=8192)) == 0
    # (whole copies of the result)
    room = L.mint_dense_workspace(dense_op(rows=64, depth=65536))
    assert room > 0 and room % (64 * 64 * 4) == 0
    # (copies of operands that are not at multiples of 16 bytes: both, or one)
    big = dict(rows=1024, cols=1001, depth=1001, x_stride=1001, w_stride=1001, out_stride=1001)
    assert L.mint_dense_workspace(dense_op(form=2, **{**big, "w_stride": 1008})) == 1001 * 2048
    assert L.mint_dense_workspace(dense_op(form=2, **{**big, "x_stride": 1024, "x": 4098})) == 1001 * 2048 + 1001 * 2016
    assert L.mint_dense_workspace(dense_op(form=2, **{**big, "x_stride": 1024, "w_stride": 1008})) == 0
    # (none of an operand of more than 4 GiB)
    far = dict(rows=1 << 20, cols=4104, depth=4097, x_stride=4097, w_stride=4104, out_stride=4104)
    assert L.mint_dense_workspace(dense_op(form=1, **far)) == 0 and L.mint_dense_workspace(dense_op(form=1, **{**far, "rows": 1 << 17})) == (1 << 17) * 8208
    assert L.mint_activation_grad_workspace(0, 5) == L.mint_activation_grad_workspace(5, 0) == 0 and L.mint_activation_grad_workspace(5, 100) == 5 * 100 * 4


@pytest.mark.parametrize("code,kw", [
    (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"d_dtype": _lib.F16}), (_lib.ERR_ARG, {"activation": 9}), (_lib.ERR_ARG, {"d": 0}), (_lib.ERR_ARG, {"z": 0}),
    (_lib.ERR_STAGING, {"workspace": 0}), (_lib.ERR_STAGING, {"workspace_bytes": 8}), (_lib.ERR_ALIGN, {"workspace": 4097}), (_lib.ERR_TOO_LARGE, {"rows": 1 << 31}),
    (_lib.OK, {"cols": 0}), (_lib.OK, {"rows": 0, "d_bias": 0})])
def test_activation_grad_refuses(code, kw):
    base = dict(d=4096, z=8192, d_z=12288, d_bias=16384, rows=5, cols=64, d_stride=64, z_stride=64, d_z_stride=64, d_dtype=_lib.F32, dtype=_lib.BF16, activation=2,
                workspace=1 << 20, workspace_bytes=1 << 20)
    assert _lib.lib().mint_activation_grad(make(_lib.ActivationGradOp, **{**base, **kw}), None) == code


def balance_op(**kw):
    return make(_lib.BalanceOp, **{**dict(logits=4096, chosen=8192, row_stride=64, tokens=5, sequences=1, experts=64, topk=2, dtype=_lib.F32), **kw})


@pytest.mark.parametrize("code,kw", [
    (_lib.ERR_ARG, {"dtype": _lib.BYTES}), (_lib.ERR_ARG, {"score": 2}), (_lib.ERR_ARG, {"experts": 0}), (_lib.ERR_ARG, {"experts": 1025}), (_lib.ERR_ARG, {"topk": 0}),
    (_lib.ERR_ARG, {"topk": 1025}), (_lib.ERR_ARG, {"logits": 0}), (_lib.ERR_ARG, {"chosen": 0}), (_lib.ERR_ARG, {"offsets": 4096, "sequences": 0}),
    (_lib.ERR_TOO_LARGE, {"tokens": 1 << 31}), (_lib.ERR_TOO_LARGE, {"offsets": 4096, "sequences": 1 << 16})])
def test_balance_refuses(code, kw):
    L = _lib.lib()
    assert L.mint_balance(balance_op(**kw), 4096, 4096, 4096, 4096, 1 << 20, 1 << 20, None) == code
    assert L.mint_balance_grad(balance_op(**kw), 4096, 4096, 4096, 0, 0, 4096, 64, None) == code
    assert L.mint_balance_workspace(balance_op(**kw)) == 0


def test_balance_refuses_results_and_workspaces():
    L = _lib.lib()
    assert L.mint_balance_workspace(balance_op(tokens=64)) == L.mint_balance_workspace(balance_op(tokens=0)) == 0           # one launch
    op = balance_op(tokens=65)
    need = L.mint_balance_workspace(op)
    assert need > 0 and L.mint_balance_workspace(balance_op(offsets=4096)) > 0
    for i in range(4):
        assert L.mint_balance(op, *(0 if j == i else 4096 for j in range(4)), 1 << 20, need, None) == _lib.ERR_ARG
        assert L.mint_balance(balance_op(), *(0 if j == i else 4096 for j in range(4)), None, 0, None) == _lib.ERR_ARG
    assert L.mint_balance(op, 4096, 4096, 4096, 4096, 1 << 20, need - 1, None) == _lib.ERR_STAGING
    assert L.mint_balance(op, 4096, 4096, 4096, 4096, None, need, None) == _lib.ERR_STAGING
    assert L.mint_balance(op, 4096, 4096, 4096, 4096, (1 << 20) + 4, need, None) == _lib.ERR_ALIGN
    assert L.mint_balance(None, 0, 0, 0, 0, None, 0, None) == L.mint_balance_grad(None, 0, 0, 0, 0, 0, 0, 0, None) == _lib.ERR_ARG
    for i in range(4):
        at = [0 if j == i else 4096 for j in range(4)]
        assert L.mint_balance_grad(balance_op(), at[0], at[1], at[2], 0, 0, at[3], 64, None) == _lib.ERR_ARG
    assert L.mint_balance_grad(balance_op(tokens=0), 0, 0, 0, 0, 0, 0, 0, None) == _lib.OK


def test_operators_take_device_tensors_only():
    x, n = torch.zeros(3, 4), Norm(torch.ones(4))
    i = torch.zeros(3, 2, dtype=torch.int32)
    found = Balance(torch.zeros(()), i, x, i[0])
    for call in (lambda: norm(x, n), lambda: norm_grad(x, x, n), lambda: join(x, x), lambda: join_grad(x, None, x, x), lambda: product(x, x),
                 lambda: activation_grad(x, x, "silu"), lambda: input_grad(x, x), lambda: weight_grad(x, x), lambda: balance(x, i),
                 lambda: balance_grad(x, x, i, found), lambda: product([1.0], x), lambda: norm(None, n)):
        with pytest.raises(TypeError, match="device tensor"):
            call()
    for call in (lambda: norm(x, n._replace(kind="none")), lambda: join(x, x, gate_by="gelu"), lambda: product(x, x, activation="softmax"), lambda: balance(x, i, score="max")):
        with pytest.raises(ValueError, match="must be"):
            call()


# ---- the oracle --------------------------------------------------------------------
def leaves(*shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_() for s in shapes]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("by,shape", [(None, (6,)), ("tanh", (4, 1)), ("sigmoid", (4, 6)), ("silu", (6,))])
def test_the_oracles_join_gradient(kind, by, shape):
    """By differences the join's definition has the gradients that torch finds, and they are the formulas'."""
    s, y, g, aw, ab, bw, bb = leaves((4, 6), (4, 6), shape, (6,), (6,), (6,), (6,))

    def both(s, y, g, aw, ab, bw, bb):
        r = 1.25 * s + 0.5 * gate64(g, by)[0] * norm64(y, aw, ab, kind, 1e-3)
        return r, norm64(r, bw, bb, kind, 1e-3)

    assert torch.autograd.gradcheck(both, (s, y, g, aw, ab, bw, bb))
    r, h = both(s, y, g, aw, ab, bw, bb)
    d, e = leaves((4, 6), (4, 6), seed=1)
    want = torch.autograd.grad((r * d).sum() + (h * e).sum(), (s, y, g, aw, ab, bw, bb))
    with torch.no_grad():
        got = join_grad64(d, e, r, y, after=(aw, ab, kind, 1e-3), gate=g, gate_by=by, scale=0.5, carry=1.25, before=(bw, bb, kind, 1e-3))
        for name, w in zip(("stream", "y", "gate", "after_weight", "after_bias", "before_weight", "before_bias"), want):
            assert torch.allclose(got[name][0], w, rtol=1e-9, atol=1e-12), name
            assert bool((got[name][1] >= got[name][0].abs() * (1 - 1e-9)).all()), name
        (dx, dw, db), _ = norm_grad64(e, s, bw, kind, 1e-3)
    s2, w2, b2 = (t.detach().requires_grad_() for t in (s, bw, bb))
    for a, b in zip((dx, dw, db), torch.autograd.grad((norm64(s2, w2, b2, kind, 1e-3) * e.detach()).sum(), (s2, w2, b2))):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-12)


def test_the_oracles_activations():
    z, = leaves((50,))
    for name in (None, "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"):
        assert torch.autograd.gradcheck(lambda t: activated64(t, name), (z,))
        step = 1e-6
        with torch.no_grad():
            want = (activated64(z + step, name) - activated64(z - step, name)) / (2 * step)
        assert torch.allclose(slope64(z, name), want, atol=1e-8)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("offsets", [None, torch.tensor([1, 4, 4, 7])])
def test_the_oracles_balance_loss(score, offsets):
    x, = leaves((8, 5))
    experts = x.detach().topk(2, 1).indices.int()
    assert torch.autograd.gradcheck(lambda t: balance64(t, experts, score, offsets, 0.3)[0], (x,))
    loss, counts, shares, there = balance64(x.detach(), experts, score, offsets, 0.0)
    assert int(counts.sum()) == 2 * int(there.sum()) and torch.allclose(shares.sum(1), (there > 0).double())
    if offsets is None:
        assert torch.allclose(loss, (counts[0] * shares[0]).sum() * 5 / 16)
