"""Attention, the norm with the residual's addition and 8-bit linear layers as a model
runs them: the attention half of a block in a serving step and in a training
pass, each stage against 64 bits on the tensors that it was given (with the bounds of
its own tests), captured and replayed, on a side stream, and again for the same bits."""
import pytest
import torch

from oracle.add_rmsnorm import fwd_bwd
from oracle.attention import packed_fwd_bwd
from oracle.int8 import linear, quantize

import test_add_rmsnorm as norm_tests
import test_attention as attention_tests
import test_int8 as int8_tests

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
HEADS, KV, D = 6, 2, 64
HIDDEN, WIDE = HEADS * D, (HEADS + 2 * KV) * D


class Block:
    """norm -> q, k, v projections -> attention -> output projection -> norm"""

    def __init__(self, dtype, backward):
        from kernels.int8 import Int8Weight

        g = torch.Generator().manual_seed(3)
        self.qkv, self.out = (Int8Weight.from_float((torch.randn(n, k, generator=g) / k ** 0.5).cuda(), backward=backward)
                              for n, k in ((WIDE, HIDDEN), (HIDDEN, HIDDEN)))
        self.norms = [(torch.rand(HIDDEN, generator=g) + 0.5).to(dtype).cuda().requires_grad_(backward) for _ in range(2)]
        self.kept = {}

    def keep(self, **tensors):
        for n, t in tensors.items():
            if isinstance(t, torch.Tensor) and t.requires_grad and not t.is_leaf:
                t.retain_grad()
            self.kept[n] = t
        return next(iter(tensors.values()))

    def split(self, qkv):
        return qkv.view(-1, HEADS + 2 * KV, D).split([HEADS, KV, KV], 1)

    def train(self, x, stream, cu):
        """(y, h) of the second norm, packed sequences."""
        from kernels.attention import forge_varlen_attention
        from kernels.int8 import int8_linear
        from kernels.rmsnorm import add_rmsnorm

        y, h = add_rmsnorm(x, stream, self.norms[0])
        self.keep(y=y), self.keep(h=h)
        qkv = self.keep(qkv=int8_linear(y, self.qkv))
        o = self.keep(o=forge_varlen_attention(*self.split(qkv), cu))
        p = self.keep(p=int8_linear(o.reshape(-1, HIDDEN), self.out))
        return add_rmsnorm(p, h, self.norms[1])

    def serve(self, x, stream, cache, cu_q, cu_k, places):
        """The same with the norms' rows in 8 bits and keys and values added to a cache [tokens, 2, KV, D]."""
        from kernels.attention import forge_varlen_attention
        from kernels.int8 import int8_linear
        from kernels.rmsnorm import add_rmsnorm_int8

        rows, h = add_rmsnorm_int8(x, stream, self.norms[0])
        qkv = self.keep(qkv=int8_linear(rows, self.qkv))
        q, k, v = self.split(qkv)
        cache[places, 0], cache[places, 1] = k, v
        o = self.keep(o=forge_varlen_attention(q, cache[:, 0], cache[:, 1], cu_q, cu_k))
        p = self.keep(p=int8_linear(o.reshape(-1, HIDDEN), self.out))
        self.kept.update(rows=rows, h=h, q=q)
        return add_rmsnorm_int8(p, h, self.norms[1])


def _draw(n, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, HIDDEN, generator=g) * std).to(dtype).cuda()


def _cpu(t):
    return t.detach().cpu()


def _check_linear(y, x, weight, what):
    ref, terms = linear(*quantize(_cpu(x)), _cpu(weight.values), _cpu(weight.scale))
    int8_tests._within(y, ref, terms, 6, what)


def _check_linear_gradient(dx, dy, weight, what):
    dy = _cpu(dy).double() * _cpu(weight.scale).double()
    ref, terms = linear(*quantize(dy), _cpu(weight.values).T, torch.ones(weight.shape[1]))
    int8_tests._within(dx, ref, terms, 6, what)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lens", [[130, 1, 77], [64], [1, 1, 2]])
def test_training(lens, dtype):
    block = Block(dtype, True)
    n = sum(lens)
    at = attention_tests._offsets(lens)
    cu = torch.tensor(at, device="cuda", dtype=torch.int32)
    x, stream = _draw(n, dtype, 0).requires_grad_(True), _draw(n, dtype, 1, 3.0).requires_grad_(True)
    dy, dh = _draw(n, dtype, 2), _draw(n, dtype, 4)
    y2, h2 = block.train(x, stream, cu)
    torch.autograd.backward((y2, h2), (dy, dh))
    kept = {k: t.detach() for k, t in block.kept.items()}
    grads = {k: t.grad for k, t in block.kept.items()}

    # forward
    w0, w1 = (_cpu(w) for w in block.norms)
    first = fwd_bwd(_cpu(x), _cpu(stream), w0, _cpu(grads["y"]), _cpu(grads["h"]), 1e-6, 0.0)
    last = fwd_bwd(_cpu(kept["p"]), _cpu(kept["h"]), w1, _cpu(dy), _cpu(dh), 1e-6, 0.0)
    assert torch.equal(_cpu(kept["h"]), first.h) and torch.equal(_cpu(h2), last.h)
    norm_tests._within(kept["y"], first.y, first.y.abs(), 100, "y")
    norm_tests._within(y2, last.y, last.y.abs(), 100, "y2")
    _check_linear(kept["qkv"], kept["y"], block.qkv, "qkv")
    _check_linear(kept["p"], kept["o"].reshape(n, HIDDEN), block.out, "p")
    q, k, v = (_cpu(t) for t in block.split(kept["qkv"]))
    ref = packed_fwd_bwd(q, k, v, _cpu(grads["o"]), at, at, D ** -0.5, True, *attention_tests._unit(dtype))
    attention_tests._within(kept["o"], ref.o, ref.o_err, "o")
    # backward
    norm_tests._within(grads["p"], last.d, last.d_terms, 200, "dp")
    _check_linear_gradient(grads["o"].reshape(n, HIDDEN), grads["p"], block.out, "do")
    for name, got in zip(("dq", "dk", "dv"), block.split(grads["qkv"])):
        attention_tests._within(got, getattr(ref, name), getattr(ref, name + "_err"), name)
    _check_linear_gradient(grads["y"], grads["qkv"], block.qkv, "dy")
    for t in (x, stream):
        norm_tests._within(t.grad, first.d, first.d_terms, 200, "dx")
    for w, r in zip(block.norms, (first, last)):
        norm_tests._within(w.grad, r.dw, r.dw_terms, 181, "dw")


def _serving(dtype=BF16, seed=0):
    """Three sequences with 200, 0 and 70 tokens before this step, room for 4 more each, and their steps' queries."""
    block = Block(dtype, False)
    held, queries, room = [200, 0, 70], [1, 3, 1], 4
    starts = attention_tests._offsets([h + room for h in held])
    g = torch.Generator().manual_seed(seed)
    cache = torch.randn(starts[-1], 2, KV, D, generator=g).to(dtype).cuda()
    return block, held, queries, starts, cache


def _step(block, held, queries, starts, cache, x, stream):
    """One step over a cache whose sequences are packed for the kernel: keys before this step's, then this step's."""
    places = torch.cat([torch.arange(s + h, s + h + n) for s, h, n in zip(starts, held, queries)]).cuda()
    live = torch.cat([torch.arange(s, s + h + n) for s, h, n in zip(starts, held, queries)]).cuda()
    packed = cache[live].clone()
    where = torch.searchsorted(live, places)
    cu_q = torch.tensor(attention_tests._offsets(queries), device="cuda", dtype=torch.int32)
    cu_k = torch.tensor(attention_tests._offsets([h + n for h, n in zip(held, queries)]), device="cuda", dtype=torch.int32)
    return block.serve(x, stream, packed, cu_q, cu_k, where), packed, cu_q, cu_k


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_serving_step(dtype):
    block, held, queries, starts, cache = _serving(dtype)
    n = sum(queries)
    x, stream = _draw(n, dtype, 5), _draw(n, dtype, 6, 3.0)
    with torch.no_grad():
        (rows, h2), packed, cu_q, cu_k = _step(block, held, queries, starts, cache, x, stream)
    kept = block.kept
    h = (_cpu(x).double() + _cpu(stream).double()).to(dtype)
    assert torch.equal(_cpu(kept["h"]), h)
    integers, _ = quantize(h.double() * _cpu(block.norms[0]).double())
    assert torch.equal(_cpu(kept["rows"].values).long(), integers)
    ref, terms = linear(integers, _cpu(kept["rows"].scale), _cpu(block.qkv.values), _cpu(block.qkv.scale))
    int8_tests._within(kept["qkv"], ref, terms, 6, "qkv")
    k, v = _cpu(packed[:, 0]), _cpu(packed[:, 1])
    q = _cpu(kept["q"])
    ref = packed_fwd_bwd(q, k, v, torch.zeros_like(q), cu_q.tolist(), cu_k.tolist(), D ** -0.5, True,
                         *attention_tests._unit(dtype))
    attention_tests._within(kept["o"], ref.o, ref.o_err, "o")
    _check_linear(kept["p"], kept["o"].reshape(n, HIDDEN), block.out, "p")
    assert torch.equal(_cpu(h2), (_cpu(kept["p"]).double() + h.double()).to(dtype))
    assert torch.equal(_cpu(rows.values).long(), quantize(_cpu(h2).double() * _cpu(block.norms[1]).double())[0])


def _capture(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def test_training_captured_and_replayed_with_other_lengths():
    """Other values and other lengths of the same total between the replays, each beside an eager pass."""
    block = Block(BF16, True)
    n = 260
    x, stream = _draw(n, BF16, 0).requires_grad_(True), _draw(n, BF16, 1, 3.0).requires_grad_(True)
    dy, dh = _draw(n, BF16, 2), _draw(n, BF16, 4)
    cu = torch.tensor([0, 100, 100, 260], device="cuda", dtype=torch.int32)
    leaves = [x, stream, *block.norms]

    def step():
        outs = block.train(x, stream, cu)
        grads = torch.autograd.grad(outs, leaves, (dy, dh))
        block.kept.clear()  # (no autograd graph of the leaves outlives its pass, as captured backward passes require)
        return (*(t.detach() for t in outs), *grads)

    graph, static = _capture(step)
    for i, offsets in enumerate(([0, 100, 100, 260], [0, 1, 200, 260], [0, 0, 260, 260], [0, 64, 128, 200])):
        with torch.no_grad():
            cu.copy_(torch.tensor(offsets, dtype=torch.int32))
            for j, t in enumerate((x, stream, dy, dh)):
                t.copy_(_draw(n, BF16, 10 * i + j))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in static]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {i}"
        torch.cuda.synchronize()


def test_serving_step_captured_and_replayed():
    """A token of each of three sequences, whose lengths grow between the replays; two captured steps whose replays
    alternate, each with a workspace of its own."""
    from kernels.attention import forge_varlen_attention
    from kernels.int8 import int8_linear
    from kernels.rmsnorm import add_rmsnorm_int8

    block = Block(BF16, False)
    total, rows = 4000, 3
    g = torch.Generator().manual_seed(8)
    keys, values = (torch.randn(total, KV, D, generator=g).to(BF16).cuda() for _ in range(2))
    cu_q = torch.arange(rows + 1, device="cuda", dtype=torch.int32)

    def make(seed):
        x, stream = _draw(rows, BF16, seed), _draw(rows, BF16, seed + 1)
        cu_k = torch.tensor([0, 1, 1300, 1500], device="cuda", dtype=torch.int32)

        def step():
            with torch.no_grad():
                a, h = add_rmsnorm_int8(x, stream, block.norms[0])
                q = int8_linear(a, block.qkv)[:, :HIDDEN].view(rows, HEADS, D)
                o, lse = forge_varlen_attention(q, keys, values, cu_q, cu_k, return_lse=True)
                b, h = add_rmsnorm_int8(int8_linear(o.reshape(rows, HIDDEN), block.out), h, block.norms[1])
                return o, lse, b.padded, b.scale, h

        return x, cu_k, step, *_capture(step)

    made = [make(20), make(30)]
    for i, offsets in enumerate(([0, 1, 1300, 1500], [0, 2, 1302, 3900], [0, 0, 0, 4000], [0, 1300, 1301, 1301])):
        for j, (x, cu_k, _, graph, _) in enumerate(made):
            cu_k.copy_(torch.tensor(offsets, dtype=torch.int32))
            x.copy_(_draw(rows, BF16, 40 + 2 * i + j))
            graph.replay()
        torch.cuda.synchronize()
        for _, _, step, _, static in made:
            got = [t.clone() for t in static]
            for a, b in zip(got, step()):
                assert torch.equal(a, b), f"replay {i}"


def test_a_side_stream_and_the_same_bits_again():
    from test_streams import _on_side_stream, _same

    block = Block(BF16, True)
    cu = torch.tensor([0, 90, 200], device="cuda", dtype=torch.int32)

    def op(x, stream, dy, dh):
        x, stream = x.detach().requires_grad_(True), stream.detach().requires_grad_(True)
        outs = block.train(x, stream, cu)
        return (*outs, *torch.autograd.grad(outs, [x, stream, *block.norms], (dy, dh)))

    def make():
        return [_draw(200, BF16, i) for i in range(4)]

    got, ref = _on_side_stream(make, op)
    _same(got, ref)
    _same(op(*make()), ref)


def test_serving_on_a_side_stream():
    from test_streams import _on_side_stream, _same

    block, held, queries, starts, cache = _serving()

    def op(x, stream):
        with torch.no_grad():
            (rows, h), *_ = _step(block, held, queries, starts, cache, x, stream)
        return rows.padded, rows.scale, h, block.kept["o"], block.kept["p"]

    got, ref = _on_side_stream(lambda: [_draw(5, BF16, i) for i in range(2)], op)
    _same(got, ref)


def _calls():
    from kernels.attention import forge_attention, forge_varlen_attention
    from kernels.int8 import Int8Weight, int8_linear, quantize_int8_rows
    from kernels.rmsnorm import add_rmsnorm, add_rmsnorm_int8

    q = torch.randn(8, 2, 64, device="cuda").to(BF16)
    cu = torch.tensor([0, 3, 8], device="cuda", dtype=torch.int32)
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    weight = Int8Weight.from_float(torch.randn(16, 64, device="cuda"), backward=True)
    return {
        "varlen q": (q, lambda t: forge_varlen_attention(t, q, q, cu)),
        "varlen k": (q, lambda t: forge_varlen_attention(q, t, q, cu)),
        "dense v": (q[None], lambda t: forge_attention(q[None], q[None], t)),
        "norm x": (x, lambda t: add_rmsnorm(t, x, w)),
        "norm residual": (x, lambda t: add_rmsnorm(x, t, w)),
        "norm weight": (w, lambda t: add_rmsnorm(x, x, t)),
        "norm rows": (x, lambda t: add_rmsnorm_int8(t, x, w)),
        "quantizer": (x, quantize_int8_rows),
        "linear": (x, lambda t: int8_linear(t, weight)),
        "bias": (w[:16], lambda t: int8_linear(x, weight, t)),
    }


@pytest.mark.parametrize("name", ["varlen q", "varlen k", "dense v", "norm x", "norm residual", "norm weight", "norm rows",
                                  "quantizer", "linear", "bias"])
def test_tangents_are_refused(name):
    from test_forward_mode import _check

    _check(*_calls()[name])


def test_second_derivatives_are_refused():
    for x, call in (_calls()[n] for n in ("varlen q", "norm x", "linear")):
        x = x.detach().requires_grad_(True)
        y = call(x)
        y = y[0] if isinstance(y, tuple) else y
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()


def test_every_entry_point_is_offered():
    import forge.kernels.attention as attention
    import forge.kernels.int8 as int8
    import forge.kernels.rmsnorm as rmsnorm
    import kernels.attention
    import kernels.int8
    import kernels.rmsnorm

    for ours, theirs, names in ((attention, kernels.attention, ("forge_attention", "forge_varlen_attention")),
                                (int8, kernels.int8, ("Int8Rows", "Int8Weight", "int8_linear", "quantize_int8_rows")),
                                (rmsnorm, kernels.rmsnorm, ("add_rmsnorm", "add_rmsnorm_int8"))):
        for n in names:
            assert getattr(ours, n) is getattr(theirs, n)
