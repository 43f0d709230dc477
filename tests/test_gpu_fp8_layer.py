"""The grouped router, the 8-bit linear layer and the 8-bit experts run together, as
a layer of a model uses them: router product, router, routed experts of the kept
tokens, shared experts, combine on the table; eager and captured in a graph."""

import pytest
import torch

from synth import make_workload
from table_moe.cache_engine.global_table import GlobalTable
from table_moe.ops import (Fp8GroupedExperts, Fp8Linear, Fp8SharedExperts, quantize_rows_fp8, quantize_weight_fp8,
                           route_experts)

pytestmark = pytest.mark.gpu

E, K, H, INTER, N_CENT = 16, 4, 512, 256, 64


def _setup(dev, n, dtype):
    wl = make_workload(5, n=n, dtype=dtype, with_slot_out=False, device=dev, hidden=H, n_experts=E, router_top_k=K,
                       n_cent=N_CENT)
    g = torch.Generator(device=dev).manual_seed(n)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=dev) * 0.05  # noqa: E731
    routed = Fp8GroupedExperts.from_weights(rnd(E, INTER, H), rnd(E, INTER, H), rnd(E, H, INTER))
    shared = Fp8SharedExperts.from_weights(rnd(2 * INTER, H), rnd(2 * INTER, H), rnd(H, 2 * INTER))
    gate = Fp8Linear(*quantize_weight_fp8(rnd(E, H)))
    table = GlobalTable(wl.centroids, wl.values, (wl.proj_vis, wl.bias_vis), (wl.proj_txt, wl.bias_txt))
    return wl, routed, shared, gate, table


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [5, 96, 1500])
def test_layer_recompute_8bit_experts(hip_device, dtype, n):
    """layer_forward_recompute with 8-bit routed and shared experts gives the bits of
    its stages called one by one, from a graph too, at every replay."""
    wl, routed, shared, _, table = _setup(hip_device, n, dtype)
    out = torch.empty_like(wl.residual)

    def layer():
        return table.layer_forward_recompute(wl.x, wl.is_vision, wl.logits, routed, wl.residual, K, 0.6, shared=shared,
                                             out=out)

    res = layer()
    torch.cuda.synchronize()
    want = {key: res[key].clone() for key in ("ids", "idx", "dist", "keep", "weights", "out")}
    kept = want["keep"].bool()
    slots = res["slot_out"].clone()
    again = torch.zeros_like(slots)
    routed.forward(wl.x, want["ids"], want["keep"], again)
    assert torch.equal(slots[kept], again[kept])
    base = shared.forward(wl.x, addend=wl.residual)
    staged = table.gather_combine(want["keep"], slots, want["weights"], want["idx"], want["dist"], base)
    assert torch.equal(want["out"], staged)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for rep in range(3):
        out.zero_()
        res["slot_out"].zero_()
        eager = shared.forward(wl.x, addend=wl.residual)  # eager work on the same weights between replays
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, base)
        for key, val in want.items():
            assert torch.equal(res[key], val), (rep, key)
        assert torch.equal(res["slot_out"][kept], slots[kept]), rep


@pytest.mark.parametrize("n", [1, 40, 700])
def test_router_to_combine(hip_device, n):
    """Router product -> router -> experts -> combine, one call after the other and
    from a graph replayed on new inputs; the combine against 64 bits."""
    wl, routed, shared, gate, table = _setup(hip_device, n, torch.bfloat16)
    x, resid = wl.x.clone(), wl.residual.clone()
    bias = torch.randn(E, generator=torch.Generator().manual_seed(1)).to(hip_device) * 0.1
    keep = torch.ones(n, dtype=torch.bool, device=hip_device)
    none = torch.zeros(n, 1, dtype=torch.long, device=hip_device)
    dist = torch.zeros(n, 1, device=hip_device)

    def run():
        rows = quantize_rows_fp8(x)
        logits = gate.forward(rows, dtype=torch.float32)
        weights, ids = route_experts(logits, K, scoring="sigmoid", bias=bias, n_groups=4, topk_groups=2,
                                     group_rule="top2", normalize_topk=True)
        slots = torch.empty(n, K, H, dtype=x.dtype, device=hip_device)
        routed.forward(x, ids, keep, slots)
        base = shared.forward(x, addend=resid)
        return logits, weights, ids, slots, base, table.gather_combine(keep, slots, weights, none, dist, base)

    logits, weights, ids, slots, base, y = (t.clone() for t in run())
    # the groups of the chosen experts: two of four
    assert int(torch.unique(ids[0] // 4).numel()) <= 2
    w = weights.double() / weights.double().sum(1, keepdim=True)
    want = base.double() + (w[:, :, None] * slots.double()).sum(1)
    # K products and sums in fp32 and weights renormalised in fp32, then half a step of bf16
    size = base.double().abs() + (w[:, :, None] * slots.double().abs()).sum(1)
    tol = (3 * K + 4) * 2.0 ** -24 * size
    tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((y.double() - want).abs() <= tol).all())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for rep in range(3):
        g = torch.Generator(device=hip_device).manual_seed(rep)
        x.copy_(torch.randn(n, H, generator=g, device=hip_device))
        resid.copy_(torch.randn(n, H, generator=g, device=hip_device))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, run()):
            assert torch.equal(a, b), rep


def test_layer_recompute_refuses_other_modules(hip_device):
    """`shared` is weights or one of the two classes; any other object with a forward
    is refused, not called."""
    wl, routed, _, _, table = _setup(hip_device, 5, torch.bfloat16)

    class Other:
        called = False

        def forward(self, hidden, out=None, addend=None):
            Other.called = True
            return out

    for other in (Other(), torch.nn.Linear(H, H)):
        with pytest.raises(TypeError):
            table.layer_forward_recompute(wl.x, wl.is_vision, wl.logits, routed, wl.residual, K, 0.6, shared=other)
    assert not Other.called


@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("n", [1, 70])
def test_which_combine_keeps_the_scale(hip_device, n, normalize):
    """combine_slots(target="orig_sum") sums the slots with the router's weights as they
    are, scale and all; gather_combine divides them by their sum."""
    from test_gpu_layer import _mode_r_manager

    wl, routed, shared, gate, table = _setup(hip_device, n, torch.bfloat16)
    mgr, _ = _mode_r_manager(hip_device, E=E, H=H)
    logits = gate.forward(wl.x).float()
    kw = dict(scoring="sigmoid", n_groups=4, topk_groups=2, group_rule="top2", normalize_topk=normalize)
    weights, ids = route_experts(logits, K, scale=2.5, **kw)
    plain, ids1 = route_experts(logits, K, **kw)
    assert torch.equal(ids, ids1)
    keep = torch.ones(n, dtype=torch.bool, device=hip_device)
    slots = torch.empty(n, K, H, dtype=wl.x.dtype, device=hip_device)
    routed.forward(wl.x, ids, keep, slots)
    base = shared.forward(wl.x, addend=wl.residual)
    every, none = (torch.full((n, K), v, dtype=torch.bool, device=hip_device) for v in (True, False))
    none_at = torch.zeros(n, K, dtype=torch.long, device=hip_device)
    got = mgr.combine_slots(weights, ids, keep, every, slots, none, none_at, residual=base, target="orig_sum")

    def check(y, w):
        want = base.double() + (w[:, :, None] * slots.double()).sum(1)
        # the coefficient: two sums of K weights, a quotient, a product; K products and
        # sums in fp32; then half a step of bf16
        size = base.double().abs() + (w[:, :, None] * slots.double().abs()).sum(1)
        tol = (3 * K + 6) * 2.0 ** -24 * size
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
        assert bool(((y.double() - want).abs() <= tol).all())

    check(got, weights.double())
    dist = torch.zeros(n, 1, device=hip_device)
    for w in (weights, plain):
        y = table.gather_combine(keep, slots, w, none_at[:, :1].contiguous(), dist, base)
        check(y, w.double() / w.double().sum(1, keepdim=True))
