"""tm_route_experts / table_moe.ops.route_experts against the definition in 64
bits: ids equal (the choice is that of 64-bit keys), weights within a few fp32
roundings (a softmax weight is a 64-bit exp over a 64-bit sum of fp32 terms, each
an expf of one ulp, 2^-23 at most, and a product rounded to 2^-24, then rounded
once itself: 2^-22 relative)."""

import numpy as np
import pytest
import torch

from fp8_ref import route
from table_moe.ops import qwen_topk_softmax, route_experts

pytestmark = pytest.mark.gpu

RTOL = 2.0 ** -22


def _check(logits, top_k, bias=None, **kw):
    got_w, got_i = route_experts(logits, top_k, bias=bias, **kw)
    ref_kw = dict(kw)
    ref_kw["normalize"] = ref_kw.pop("normalize_topk", False)
    if ref_kw.get("topk_groups") is None:
        ref_kw["topk_groups"] = ref_kw.get("n_groups", 1)
    want_w, want_i = route(logits.double().cpu().numpy(), top_k, bias=None if bias is None else bias.cpu().numpy(),
                           **ref_kw)
    assert got_w.dtype == torch.float32 and got_i.dtype == torch.long
    np.testing.assert_array_equal(got_i.cpu().numpy(), want_i)
    np.testing.assert_allclose(got_w.cpu().double().numpy(), want_w, rtol=RTOL, atol=1e-37)
    return got_w, got_i


def _logits(seed, n, e, dev, dtype=torch.float32, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(n, e, generator=g)).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,e,top_k,groups,keep,rule,scoring,bias", [
    (1, 256, 8, 8, 4, "top2", "sigmoid", True),
    (37, 256, 8, 8, 4, "top2", "sigmoid", True),
    (33, 160, 6, 8, 3, "max", "softmax", False),
    (5, 64, 6, 1, 1, "max", "softmax", True),
    (130, 64, 6, 1, 1, "max", "sigmoid", False),
    (9, 72, 4, 3, 2, "top2", "softmax", True),
    (3, 1024, 32, 64, 5, "top2", "sigmoid", False),
    (6, 300, 17, 4, 1, "max", "sigmoid", True),
    (4, 1, 1, 1, 1, "max", "softmax", False),
    (4, 7, 7, 7, 7, "top2", "sigmoid", True),  # groups of one expert
])
def test_matches_definition(hip_device, dtype, n, e, top_k, groups, keep, rule, scoring, bias):
    x = _logits(n * 7 + e, n, e, hip_device, dtype)
    b = _logits(5, 1, e, hip_device, spread=0.1)[0] if bias else None
    for norm, scale in ((False, 1.0), (True, 2.5)):
        _check(x, top_k, b, scoring=scoring, n_groups=groups, topk_groups=keep, group_rule=rule, normalize_topk=norm,
               scale=scale)


@pytest.mark.parametrize("scoring,bias,rule", [("sigmoid", True, "top2"), ("softmax", True, "max"),
                                               ("softmax", False, "max"), ("sigmoid", False, "top2")])
@pytest.mark.parametrize("e,groups,keep,top_k", [(256, 8, 4, 8), (1024, 2, 1, 32), (60, 20, 10, 12), (64, 64, 32, 31),
                                                 (99, 3, 1, 9), (500, 4, 2, 16), (112, 7, 3, 6)])
def test_few_groups_stay(hip_device, e, groups, keep, top_k, scoring, bias, rule):
    """At most half of the experts open: logits with many equals, experts that are
    not available (whole groups of them in some rows)."""
    x = _logits(e, 41, e, hip_device)
    x[:20] = (x[:20] * 2).round() / 2
    x[5:15][torch.rand(10, e, generator=torch.Generator().manual_seed(3)).to(hip_device) < 0.4] = float("-inf")
    x[3, : e // groups] = float("-inf")
    x[4, e // groups:] = float("nan")
    b = _logits(5, 1, e, hip_device, spread=0.1)[0] if bias else None
    _check(x, top_k, b, scoring=scoring, n_groups=groups, topk_groups=keep, group_rule=rule, normalize_topk=True)


def test_softmax_matches_topk_softmax(hip_device):
    x = _logits(3, 65, 128, hip_device)
    w, i = route_experts(x, 8, normalize_topk=True)
    w0, i0 = qwen_topk_softmax(x, 8, normalize_topk=True)
    assert torch.equal(i, i0)
    torch.testing.assert_close(w, w0, rtol=1e-5, atol=0)


def test_ties_go_to_the_lower_id(hip_device):
    x = torch.zeros(3, 96, device=hip_device)
    x[1, 5::7] = 1.0
    x[2] = torch.arange(96, device=hip_device) // 10 * 0.5
    b = torch.zeros(96, device=hip_device)
    for bias in (None, b):
        for groups, keep, rule in ((1, 1, "max"), (8, 3, "max"), (8, 3, "top2")):
            for scoring in ("softmax", "sigmoid"):
                _check(x, 9, bias, scoring=scoring, n_groups=groups, topk_groups=keep, group_rule=rule)


def test_keys_that_differ_past_fp32(hip_device):
    # sigmoid(l) + b of neighbours differ by about 1e-9: equal or swapped in fp32
    n, e = 64, 64
    g = torch.Generator().manual_seed(9)
    x = torch.randn(n, e, generator=g)
    s = torch.sigmoid(x[0].double())
    b = (0.75 - s).float()  # row 0: every key is 0.75 up to b's rounding
    x[:] = x[0]
    _check(x.to(hip_device), 16, b.to(hip_device), scoring="sigmoid")
    _check(x.to(hip_device), 16, b.to(hip_device), scoring="sigmoid", n_groups=8, topk_groups=4, group_rule="top2")


def test_saturated_logits_keep_their_order(hip_device):
    # sigmoid and softmax round to equal scores; the logits still order the experts
    x = torch.linspace(60.0, 90.0, 64)[torch.randperm(64, generator=torch.Generator().manual_seed(1))][None]
    _check(x.to(hip_device), 8, scoring="sigmoid")
    y = torch.linspace(-3e4, 0.0, 64)[torch.randperm(64, generator=torch.Generator().manual_seed(2))][None]
    _check(y.to(hip_device), 8, scoring="softmax")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
def test_masked_experts(hip_device, scoring, bias):
    e = 64
    x = _logits(11, 8, e, hip_device)
    x[1, ::2] = float("-inf")
    x[2, 3:] = float("-inf")          # fewer available than chosen
    x[3] = float("-inf")              # none
    x[4, 7] = float("nan")
    x[5, 9] = float("inf")
    x[5, 40] = float("inf")
    x[6, :32] = float("-inf")
    x[6, 33] = float("nan")
    x[7] = float("nan")
    b = None
    if bias:
        b = _logits(12, 1, e, hip_device, spread=0.3)[0]
        b[0], b[1], b[2] = float("-inf"), float("nan"), 5.0
    for groups, keep, rule in ((1, 1, "max"), (8, 2, "max"), (8, 2, "top2"), (32, 4, "top2")):
        for norm in (False, True):
            w, i = _check(x, 6, b, scoring=scoring, n_groups=groups, topk_groups=keep, group_rule=rule,
                          normalize_topk=norm)
            assert torch.isfinite(w).all() and int(i.min()) >= 0 and int(i.max()) < e
            assert float(w[3].abs().max()) == 0.0 and float(w[7].abs().max()) == 0.0


def test_strides_and_empty(hip_device):
    x = _logits(4, 20, 100, hip_device)
    wide = torch.full((20, 130), 9.0, device=hip_device)
    wide[:, 10:110] = x
    view = wide[:, 10:110]            # row stride 130, rows not 16-byte aligned
    w, i = route_experts(view, 5, scoring="sigmoid")
    w0, i0 = route_experts(x, 5, scoring="sigmoid")
    assert torch.equal(w, w0) and torch.equal(i, i0)
    w, i = route_experts(x.t().contiguous().t(), 5, scoring="sigmoid")
    assert torch.equal(w, w0) and torch.equal(i, i0)
    w, i = route_experts(x[:0], 5)
    assert w.shape == (0, 5) and i.shape == (0, 5)


def test_one_row_for_all_tokens(hip_device):
    """Row stride 0, and one expert."""
    x = _logits(4, 1, 100, hip_device)
    w0, i0 = route_experts(x, 5)
    w, i = route_experts(x.expand(37, 100), 5)
    assert torch.equal(w, w0.expand(37, 5)) and torch.equal(i, i0.expand(37, 5))
    w, i = route_experts(x[:, :1].expand(9, 1), 1)
    assert bool((w == 1).all()) and bool((i == 0).all())
    w, i = route_experts(_logits(5, 9, 4, hip_device)[:, 1:2], 1)   # a column
    assert bool((w == 1).all()) and bool((i == 0).all())


def test_other_stream_and_graph(hip_device):
    x = _logits(6, 50, 256, hip_device)
    b = _logits(7, 1, 256, hip_device, spread=0.1)[0]
    kw = dict(scoring="sigmoid", n_groups=8, topk_groups=4, group_rule="top2", normalize_topk=True, scale=2.5)
    want = route_experts(x, 8, bias=b, **kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = route_experts(x, 8, bias=b, **kw)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = route_experts(x, 8, bias=b, **kw)
    for seed in (21, 22, 23):
        x.copy_(_logits(seed, 50, 256, hip_device))
        graph.replay()
        want = route_experts(x, 8, bias=b, **kw)
        torch.cuda.synchronize()
        assert torch.equal(cap[0], want[0]) and torch.equal(cap[1], want[1])


def test_refusals(hip_device):
    x = _logits(1, 4, 64, hip_device)
    for kw in (dict(top_k=0), dict(top_k=65), dict(top_k=33), dict(top_k=4, scoring="tanh"),
               dict(top_k=4, n_groups=5), dict(top_k=4, n_groups=8, topk_groups=9),
               dict(top_k=9, n_groups=8, topk_groups=1), dict(top_k=4, n_groups=8, topk_groups=0),
               dict(top_k=4, group_rule="sum"), dict(top_k=4, scale=float("nan"))):
        with pytest.raises(ValueError):
            route_experts(x, **kw)
    with pytest.raises(ValueError):
        route_experts(x[0], 4)
    with pytest.raises(ValueError):
        route_experts(x, 4, bias=torch.zeros(63, device=hip_device))
    with pytest.raises(ValueError):
        route_experts(x.double(), 4)
    with pytest.raises(ValueError):
        route_experts(torch.zeros(2, 1025, device=hip_device), 4)
    with pytest.raises(RuntimeError):
        route_experts(x.cpu(), 4)


def _near_ties(seed, e, scoring, rows=5):
    """Logits and a bias that makes every key of row 0 equal up to the bias's own
    rounding to fp32 (gaps of 1e-11 to 1e-8); row r: row 0's logits moved by r / 2,
    whose softmax scores are row 0's up to a rounding."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(1, e, generator=g)
    s = torch.softmax(x[0].double(), 0) if scoring == "softmax" else torch.sigmoid(x[0].double())
    bias = (0.75 - s).float()
    return x + 0.5 * torch.arange(rows)[:, None], bias


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,top_k,groups,keep,rule", [
    (64, 16, 1, 1, "max"), (256, 8, 1, 1, "max"), (64, 32, 1, 1, "max"), (64, 6, 8, 4, "top2"), (256, 8, 8, 4, "top2"),
    (256, 8, 8, 3, "max"), (72, 9, 3, 2, "top2"), (512, 16, 4, 2, "max"),
])
def test_near_ties_of_many_draws(hip_device, scoring, e, top_k, groups, keep, rule):
    """The order of keys that only 64 bits tell apart, another bias in every call.  A
    softmax score's sum of e terms is within e 2^-53 of its size on either side, and a
    key of under 1 takes a few roundings of 2^-53 more: draws with two keys nearer
    than that are left out."""
    taken = 0
    for seed in range(40):
        x, bias = _near_ties(1000 * e + seed, e, scoring)
        z = x.double()
        score = torch.softmax(z, 1) if scoring == "softmax" else torch.sigmoid(z)
        error = (8 + (e * float(score.max()) if scoring == "softmax" else 0)) * 2.0 ** -52
        if float((score + bias.double()).sort(1).values.diff(dim=1).min()) < error:
            continue
        taken += 1
        _check(x.to(hip_device), top_k, bias.to(hip_device), scoring=scoring, n_groups=groups, topk_groups=keep,
               group_rule=rule)
    assert taken >= 20


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [16.0, 1e3, 1e4, 1e6, 1e30])
def test_group_values_of_large_biases_that_cancel(hip_device, scoring, size):
    """A group's two best keys of opposite sign: their sum in fp32 keeps little of
    the scores, in 64 bits it does."""
    for seed in range(4):
        e, groups = 48, 12
        x = _logits(seed, 401, e, hip_device)
        b = torch.full((groups, 4), -4 * size)
        b[:, seed % 3], b[:, 3] = size, -size
        _check(x, 8, b.reshape(-1).to(hip_device), scoring=scoring, n_groups=groups, topk_groups=5, group_rule="top2")


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("rule", ["max", "top2"])
def test_group_values_past_fp32(hip_device, scoring, rule):
    """Sums of two keys over fp32's largest number, under its lowest, and infinite
    biases, beside groups that are not available."""
    big, inf = 3.4e38, float("inf")
    x = _logits(3, 9, 32, hip_device)
    for rows in ([[big, 1e38], [big, 2e38], [big, big], [3e38, 3e38], [0, 0], [1, 1], [2, 2], [3, 3]],
                 [[-big, -big], [-inf, -inf], [-big, -2e38], [-3e38, -3e38], [-inf, -big], [-2e38, -big],
                  [-inf, -inf], [-1e38, -big]],
                 [[inf, inf], [inf, 1], [inf, -big], [big, big], [2e38, 2e38], [inf, inf], [5, 5], [5.0000005, 5]],
                 [[-inf, -inf], [-big, -big], [-inf, -inf], [-inf, -inf], [-2e38, -2e38], [-inf, -inf], [-inf, -inf],
                  [-inf, -inf]]):
        b = torch.full((8, 4), -inf)
        b[:, 1:3] = torch.tensor(rows)
        for keep in (1, 2, 3, 5):
            _check(x, 4, b.reshape(-1).to(hip_device), scoring=scoring, n_groups=8, topk_groups=keep, group_rule=rule)
