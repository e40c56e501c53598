"""The learning operators together and beside the strict path: a distillation step of a network with a
normalised layer, the guarded chain, and the Python layer's refusals."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import learn_util as lu
from gpu_util import status_word

pytestmark = pytest.mark.gpu


def _teacher(provider, x, w1, w2, k):
    """The frozen network: two 8-bit products, its top logits."""
    def layer(v, w):
        codes, scales = provider.block_quantize(v)
        return provider.block_matmul(codes, scales, *provider.block_quantize(w, 128), dtype=torch.float32)

    top, at = layer(layer(x, w1).relu(), w2).topk(k, dim=1)
    return at, top


def test_a_distillation_step(provider):
    """Teacher by 8-bit products; student = strict MatMul, group norm with SiLU, strict MatMul; the loss, its
    gradient, the backward pass with strict MatMuls, SGD.  The loss and all gradients are compared with the same
    step in 64 bits on the same teacher entries.  Tolerance: each value passes three sums of at most 512 binary32
    terms in index order (511 u of the magnitudes, each) and the operators' own, smaller errors; u = 2^-24, the
    magnitudes' sums are below 40 times the largest gradient here, so 3 * 512 * u * 40 = 3.7e-3 of it bounds all
    (observed about 1e-6)."""
    gen = torch.Generator().manual_seed(1)
    rows, wide, hidden, vocab, k, t = 96, 64, 128, 512, 16, 2.0

    def normal(*shape):
        return torch.randn(shape, generator=gen).cuda()

    x, tw1, tw2 = normal(rows, wide), normal(hidden, wide) / 8, normal(vocab, hidden) / 3
    at, top = _teacher(provider, x, tw1, tw2, k)
    w1, w2, gw, gb = normal(wide, hidden) / 8, normal(hidden, vocab) / 11, 1 + normal(hidden) / 5, normal(hidden) / 5
    up = torch.full((1,), 1.0 / rows, device="cuda")
    status = provider.new_status(9)
    words = [status[i:i + 1] for i in range(9)]

    a = provider.strict_matmul(x, w1, policy=2, status=words[0])
    y, stats = provider.group_norm(a, 8, gw, gb, activation="silu", status=words[1])
    z = provider.strict_matmul(y, w2, policy=2, status=words[2])
    loss, _, dz = provider.distill_loss_step(z, at, top, upstream=up, temperature=t, status=words[3])
    dw2 = provider.strict_matmul(y, dz, transpose_left=True, policy=2, status=words[4])
    dy = provider.strict_matmul(dz, w2, transpose_right=True, policy=2, status=words[5])
    da, dgw, dgb = provider.group_norm_backward(a, dy, 8, stats, gw, gb, activation="silu", status=words[6])
    dw1 = provider.strict_matmul(x, da, transpose_left=True, policy=2, status=words[7])
    new = provider.strict_sgd(w1, dw1, 0.5, policy=2, status=words[8])
    assert bool((status == -1).all())

    p = [v.double().requires_grad_() for v in (w1, w2, gw, gb)]
    a64 = x.double() @ p[0]
    v = a64.reshape(rows, 8, hidden // 8)
    mean = v.mean(dim=2, keepdim=True)
    var = ((v - mean) ** 2).mean(dim=2, keepdim=True)
    h = ((v - mean) / torch.sqrt(var + float(np.float32(1e-5)))).reshape(rows, hidden) * p[2] + p[3]
    y64 = h * torch.sigmoid(h)
    lq = torch.log_softmax(y64 @ p[1] / t, dim=1)
    lp = torch.log_softmax(top.double() / t, dim=1)
    rows64 = t * t * (lp.exp() * (lp - lq.gather(1, at))).sum(dim=1)
    (rows64.sum() / rows).backward()
    for got, want in [(loss, rows64)] + list(zip((dw1, dw2, dgw, dgb), (q.grad for q in p))):
        lu.within(got, want.detach(), 3.7e-3 * float(want.detach().abs().max()))
    want = w1.double() - 0.5 * dw1.double()
    lu.within(new, want, 2 * lu.u(torch.float32) * (w1.double().abs() + dw1.double().abs()))


def test_teacher_for_one_row_is_the_batch_s(provider):
    """A single row through the quantised layers gives the batch's row (each within its rounding)."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn((200, 384), generator=gen).cuda()
    w = torch.randn((700, 384), generator=gen).cuda()
    codes, scales = provider.block_quantize(w, 128)
    a, sa = provider.block_quantize(x)
    batch = provider.block_matmul(a, sa, codes, scales, dtype=torch.float32)
    for row in (0, 57, 199):
        one, s1 = provider.block_quantize(x[row:row + 1])
        assert torch.equal(one.view(torch.uint8), a[row:row + 1].view(torch.uint8)) and torch.equal(s1, sa[row:row + 1])
        single = provider.block_matmul(one, s1, codes, scales, dtype=torch.float32)
        size = (one.float() * s1.repeat_interleave(128, 1)[:, :384]).abs() @ \
            (codes.float() * scales.repeat_interleave(128, 0)[:700].repeat_interleave(128, 1)).abs().t()
        lu.within(single, batch[row:row + 1], 2 * 134 * lu.u(torch.float32) * size.double())


def test_guarded_chain(provider):
    """Each call as a stage: admitted while nothing faulted, the same bits; skipped after a fault, its
    outputs untouched."""
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((6, 5, 32), generator=gen).cuda()
    dy = torch.randn((6, 5, 32), generator=gen).cuda()
    z = torch.randn((6, 400), generator=gen).cuda()
    top, at = torch.randn((6, 400), generator=gen).cuda().topk(4, dim=1)
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    y0, st0 = provider.group_norm(x, 4, w, b, activation="relu")
    g0 = provider.group_norm_backward(x, dy, 4, st0, w, b, activation="relu")
    l0, s0 = provider.distill_loss(z, at, top)
    d0 = provider.distill_loss_backward(z, at, top, s0)
    q0, qs0 = provider.block_quantize(z)
    w0, ws0 = provider.block_quantize(torch.randn((70, 400), generator=gen).cuda(), 128)
    p0 = provider.block_matmul(q0, qs0, w0, ws0)

    def run(first):
        c = provider.GuardedChain(8).reset()
        outs = {}
        provider.checked_relu(first, chain=c.stage(0))
        outs["y"], st = torch.full_like(x, 7), torch.full_like(st0, 7)
        provider.group_norm(x, 4, w, b, activation="relu", out=outs["y"], stats=st, chain=c.stage(1))
        outs["dx"], outs["dw"], outs["db"] = torch.full_like(x, 7), torch.full_like(w, 7), torch.full_like(b, 7)
        provider.group_norm_backward(x, dy, 4, st, w, b, activation="relu", dx=outs["dx"], dweight=outs["dw"],
                                     dbias=outs["db"], chain=c.stage(2))
        outs["loss"], stats = torch.full_like(l0, 7), torch.full_like(s0, 7)
        provider.distill_loss(z, at, top, loss=outs["loss"], stats=stats, chain=c.stage(3))
        outs["dz"] = torch.full_like(z, 7)
        provider.distill_loss_backward(z, at, top, stats, gradient=outs["dz"], chain=c.stage(4))
        outs["loss2"], outs["dz2"] = torch.full_like(l0, 7), torch.full_like(z, 7)
        provider.distill_loss_step(z, at, top, loss=outs["loss2"], stats=torch.empty_like(stats), gradient=outs["dz2"],
                                   chain=c.stage(5))
        codes, scales = torch.full((6, 400), 7, dtype=torch.uint8, device="cuda"), torch.full_like(qs0, 7)
        provider.block_quantize(z, codes=codes, scales=scales, chain=c.stage(6))
        outs["scales"], outs["codes"] = scales, codes
        outs["p"] = torch.full_like(p0, 7)
        provider.block_matmul(codes, scales, w0, ws0, out=outs["p"], chain=c.stage(7))
        return c, outs

    chain, outs = run(torch.zeros(4, device="cuda"))
    assert chain.validate([4, 960, 960 + 64, 6, 6, 6, 2400, 420])[0] == "succeeded"
    want = {"y": y0, "dx": g0[0], "dw": g0[1], "db": g0[2], "loss": l0, "dz": d0, "loss2": l0, "dz2": d0, "scales": qs0,
            "codes": q0.view(torch.uint8), "p": p0}
    for name, v in want.items():
        assert torch.equal(outs[name], v), name
    chain, outs = run(torch.full((4,), math.nan, device="cuda"))
    outcome, stage, _ = chain.validate()
    assert (outcome, stage) == ("fault", 0)
    assert all(bool((v == 7).all()) for v in outs.values())


def test_guarded_chain_stops_at_a_learning_fault(provider):
    x = torch.randn((4, 32), device="cuda")
    x[2, 1] = math.nan
    c = provider.GuardedChain(2).reset()
    provider.group_norm(x, 4, chain=c.stage(0))
    out = torch.full((4, 32), 7.0, device="cuda")
    provider.group_norm(torch.zeros_like(x), 4, out=out, chain=c.stage(1))
    assert c.validate([128, 128]) == ("fault", 0, ((2 * 32) << 3) | 5)
    assert bool((out == 7).all())


def test_first_calls_may_be_captured(provider):
    """A process whose very first call of each operator is inside a graph capture."""
    code = """
import importlib, torch
pcu = importlib.import_module("fusion-pcu_b200")
torch.manual_seed(0)
x = torch.randn((8, 900, 64), device="cuda"); z = torch.randn((3, 60000), device="cuda"); top, at = z.topk(8, dim=1)
v = torch.randn((70, 512), device="cuda"); status = pcu.new_status()
torch.cuda.synchronize()

def calls():
    y, stats = pcu.group_norm(x, 8, activation="gelu", status=status)
    dx = pcu.group_norm_backward(x, x, 8, stats, activation="gelu", status=status)[0]
    g = pcu.distill_loss_step(z, at, top, status=status)[2]
    codes, scales = pcu.block_quantize(v, status=status)
    w, ws = pcu.block_quantize(v, 128, status=status)
    return y, dx, g, pcu.block_matmul(codes, scales, w, ws, status=status), pcu.block_matmul(codes[:4], scales[:4], w, ws, status=status)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, calls())) and int(status[0]) == -1
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stdout + run.stderr


def test_two_streams_at_once(provider):
    """The operators keep no state between calls: the same calls on two streams at once, many times, give
    the bits of one."""
    gen = torch.Generator().manual_seed(4)
    x = torch.randn((4, 2000, 64), generator=gen).cuda()
    z = torch.randn((50, 70000), generator=gen).cuda()
    top, at = z.topk(8, dim=1)
    v = torch.randn((300, 512), generator=gen).cuda()
    w, ws = provider.block_quantize(torch.randn((500, 512), generator=gen).cuda(), 128)

    def calls(stream=None):
        y, stats = provider.group_norm(x, 8, activation="silu", stream=stream)
        dx = provider.group_norm_backward(x, x, 8, stats, activation="silu", stream=stream)[0]
        g = provider.distill_loss_step(z, at, top, stream=stream)
        codes, scales = provider.block_quantize(v, stream=stream)
        return (y, dx) + g + (provider.block_matmul(codes, scales, w, ws, stream=stream),
                              provider.block_matmul(codes[:8], scales[:8], w, ws, stream=stream))

    want = calls()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[calls(s) for s in streams] for _ in range(5)]
    torch.cuda.synchronize()
    for both in got:
        for outs in both:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_empty_stages_decide(provider):
    c = provider.GuardedChain(3).reset()
    provider.group_norm(torch.empty((0, 8), device="cuda"), 2, chain=c.stage(0))
    provider.distill_loss(torch.empty((0, 8), device="cuda"), torch.empty((0, 2), dtype=torch.int64, device="cuda"),
                          torch.empty((0, 2), device="cuda"), chain=c.stage(1))
    provider.block_quantize(torch.empty((0, 8), device="cuda"), chain=c.stage(2))
    assert c.validate()[0] == "succeeded"


def test_python_refusals(provider):
    x = torch.randn((4, 6, 8), device="cuda")
    f = torch.float8_e4m3fn
    bad = [
        (ValueError, lambda: provider.group_norm(x.cpu(), 2)), (ValueError, lambda: provider.group_norm(x, 3)),
        (ValueError, lambda: provider.group_norm(x, 0)), (ValueError, lambda: provider.group_norm(x, 2, activation="tanh")),
        (ValueError, lambda: provider.group_norm(x[0, 0], 2)), (TypeError, lambda: provider.group_norm(x.int(), 2)),
        (ValueError, lambda: provider.group_norm(x.transpose(1, 2), 2)),
        (TypeError, lambda: provider.group_norm(x, 2, torch.ones(8, device="cuda").half())),
        (ValueError, lambda: provider.group_norm(x, 2, torch.ones(7, device="cuda"))),
        (ValueError, lambda: provider.group_norm(x, 2, torch.ones(8))),
        (ValueError, lambda: provider.group_norm(x, 2, out=torch.empty((4, 6, 9), device="cuda"))),
        (provider.ProviderFailure, lambda: provider.group_norm(x[:, :1].expand(4, 6, 8), 2)),
        (provider.ProviderFailure, lambda: provider.group_norm(x, 2, eps=-1.0)),
        (ValueError, lambda: provider.group_norm_backward(x, x[:, :5], 2, torch.ones((4, 2, 2), device="cuda"))),
        (ValueError, lambda: provider.group_norm_backward(x, x, 2, torch.ones((4, 3, 2), device="cuda"))),
    ]
    z = torch.randn((3, 50), device="cuda")
    top, at = z.topk(2, dim=1)
    bad += [
        (TypeError, lambda: provider.distill_loss(z, at.int(), top)), (ValueError, lambda: provider.distill_loss(z, at[:2], top)),
        (ValueError, lambda: provider.distill_loss(z, at, top[:, :1].contiguous())),
        (TypeError, lambda: provider.distill_loss(z, at, top.half())), (ValueError, lambda: provider.distill_loss(z.t(), at, top)),
        (ValueError, lambda: provider.distill_loss(z[0], at, top)),
        (provider.ProviderFailure, lambda: provider.distill_loss(z, at, top, temperature=0.0)),
        (ValueError, lambda: provider.distill_loss(z, at, top, row_weights=torch.ones(2, device="cuda"))),
        (ValueError, lambda: provider.distill_loss_step(z, at, top, upstream=torch.ones(2, device="cuda"))),
        (ValueError, lambda: provider.distill_loss_step(z, at, top, gradient=torch.empty((3, 51), device="cuda"))),
        (ValueError, lambda: provider.distill_loss(z, torch.zeros((3, 1025), dtype=torch.int64, device="cuda"),
                                                   torch.zeros((3, 1025), device="cuda"))),
        (TypeError, lambda: provider.block_quantize(z.double())), (ValueError, lambda: provider.block_quantize(z, 64)),
        (ValueError, lambda: provider.block_quantize(z, codes=torch.empty((3, 49), dtype=f, device="cuda"))),
        (TypeError, lambda: provider.block_quantize(z, codes=torch.empty((3, 50), device="cuda"))),
    ]
    q, s = provider.block_quantize(z)
    w, ws = provider.block_quantize(z, 128)
    bad += [
        (ValueError, lambda: provider.block_matmul(q, s, w[:, :49], ws)), (ValueError, lambda: provider.block_matmul(q, ws, w, ws)),
        (TypeError, lambda: provider.block_matmul(z, s, w, ws)), (TypeError, lambda: provider.block_matmul(q, s.double(), w, ws)),
        (ValueError, lambda: provider.block_matmul(q, s, w, ws, out=torch.empty((3, 4), device="cuda"))),
        (ValueError, lambda: provider.block_matmul(q, s, w, ws, dtype=torch.float64)),
    ]
    for error, call in bad:
        with pytest.raises(error):
            call()
    # arguments by name, the first one too
    assert torch.equal(provider.group_norm(x=x, groups=2)[0], provider.group_norm(x, 2)[0])
    assert status_word(provider.new_status()) == provider.STATUS_OK


def _chained(provider, x, w, ws, logits, at, top, after=lambda: None):
    """Calls that each need the one before, with buffers used again at once: an early start shows."""
    codes = scales = norm = None
    for _ in range(12):
        codes, scales = provider.block_quantize(x, codes=codes, scales=scales)
        after()
        y = provider.block_matmul(codes, scales, w, ws, dtype=torch.float32)
        after()
        norm, stats = provider.group_norm(y, 4, activation="silu", out=norm)
        after()
        dx, _, _ = provider.group_norm_backward(y, norm, 4, stats, activation="silu", dx=y)
        after()
        _, row, gradient = provider.distill_loss_step(logits, at, top, upstream=dx[:, 0].contiguous(), gradient=logits)
        after()
        x = provider.group_norm(dx + gradient[:, :dx.shape[1]], 4, out=x)[0]
        after()
    return x, gradient


@pytest.mark.parametrize("rows", [3, 200])
def test_calls_keep_the_order_of_their_stream(provider, rows):
    """The same bits whether each call has ended before the next is made, follows at once, or is replayed in a graph
    with a fork and a join between them."""
    gen = torch.Generator().manual_seed(rows)
    x0 = torch.randn((rows, 512), generator=gen).cuda()
    z0 = torch.randn((rows, 20000), generator=gen).cuda()
    top, at = z0.topk(8, dim=1)
    w, ws = provider.block_quantize(torch.randn((512, 512), generator=gen).cuda(), 128)
    want = _chained(provider, x0.clone(), w, ws, z0.clone(), at, top, torch.cuda.synchronize)
    got = _chained(provider, x0.clone(), w, ws, z0.clone(), at, top)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    x, z = x0.clone(), z0.clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        aside, _ = provider.group_norm(x0, 4, stream=side)
        out = _chained(provider, x, w, ws, z, at, top)
        torch.cuda.current_stream().wait_stream(side)
        both = provider.group_norm(out[0] + aside, 4)[0]
    for _ in range(3):
        x.copy_(x0), z.copy_(z0)
        graph.replay()
    assert torch.equal(want[0], out[0]) and torch.equal(want[1], out[1])
    assert torch.equal(both, provider.group_norm(want[0] + provider.group_norm(x0, 4)[0], 4)[0])
