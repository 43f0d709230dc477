"""Derivatives of rotate_positions on the CPU: the kernel's launch is replaced by the same rotation in torch, so that what
is tested is the path around it (which calls have derivatives, and of what)."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from table_moe.ops import rotary

N_TOK, H, KV, D = 5, 3, 2, 8
SECTIONS = (2, 1, 1)


def turn(x, positions, inv_freq, inverse):
    axis = torch.tensor([0, 0, 1, 2])
    angle = (positions[axis].double() * inv_freq.double()[:, None]).T[:, None] * (-1 if inverse else 1)
    c, s = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    a, b = x[..., :4], x[..., 4:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.fixture
def on_host(monkeypatch):
    def run(q, k, positions, inv_freq, sections, interleaved, adjacent, inverse, q_out, k_out, dev):
        assert sections == SECTIONS and not interleaved and not adjacent
        with torch.no_grad():  # (a launch sees numbers alone: no tangents either)
            for x, out in ((q, q_out), (k, k_out)):
                if x is not None:
                    out.copy_(turn(fwd.unpack_dual(x).primal, positions, fwd.unpack_dual(inv_freq).primal, inverse))

    monkeypatch.setattr(rotary, "_run", run)
    monkeypatch.setattr(rotary.N, "require_hip", lambda *t: torch.device("cpu"))


@pytest.fixture
def data():
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(0, 50, (3, N_TOK), generator=g)
    inv = torch.rand(4, generator=g)
    mk = lambda h: torch.randn(N_TOK, h, D, generator=g)  # noqa: E731
    return pos, inv, mk(H), mk(KV), mk(H), mk(KV)


@pytest.mark.parametrize("inverse", [False, True])
def test_forward_mode(on_host, data, inverse):
    pos, inv, q, k, tq, tk = data
    call = lambda a, b: rotary.rotate_positions(a, b, pos, inv, SECTIONS, inverse=inverse)  # noqa: E731
    with fwd.dual_level():
        y, z = call(fwd.make_dual(q, tq), fwd.make_dual(k, tk))
        for out, x, t in ((y, q, tq), (z, k, tk)):
            p, tangent = fwd.unpack_dual(out)
            assert torch.equal(p, turn(x, pos, inv, inverse)) and torch.equal(tangent, turn(t, pos, inv, inverse))
        y, z = call(q, fwd.make_dual(k, tk))  # one of them alone
        t = fwd.unpack_dual(y).tangent
        assert t is None or not bool(t.any())
        assert torch.equal(fwd.unpack_dual(z).tangent, turn(tk, pos, inv, inverse))
        y, none = call(fwd.make_dual(q, tq), None)
        assert none is None and torch.equal(fwd.unpack_dual(y).tangent, turn(tq, pos, inv, inverse))
        with torch.no_grad():  # tangents flow there, too
            assert torch.equal(fwd.unpack_dual(call(fwd.make_dual(q, tq), k)[0]).tangent, turn(tq, pos, inv, inverse))
        assert fwd.unpack_dual(call(q, k)[0]).tangent is None
    assert torch.equal(call(q, k)[0], turn(q, pos, inv, inverse))


def test_forward_over_reverse(on_host, data):
    """The tangent of a gradient: d/dt of the gradient of sum(w y^3) at q + t tq, and the other way round."""
    pos, inv, q, k, tq, _ = data
    call = lambda a: rotary.rotate_positions(a, None, pos, inv, SECTIONS)[0]  # noqa: E731
    y, ty = turn(q, pos, inv, False), turn(tq, pos, inv, False)
    want = turn(6 * y * ty, pos, inv, True)
    with fwd.dual_level():
        x = fwd.make_dual(q.clone().requires_grad_(), tq)
        grad, = torch.autograd.grad((call(x) ** 3).sum(), x, create_graph=True)
        assert torch.allclose(fwd.unpack_dual(grad).tangent, want, rtol=1e-5, atol=1e-5)
    a = q.clone().requires_grad_()
    with fwd.dual_level():
        out, tangent = fwd.unpack_dual(call(fwd.make_dual(a, tq)) ** 3)
        back, = torch.autograd.grad(tangent.sum(), a)
    assert torch.allclose(back, want, rtol=1e-5, atol=1e-5)


def test_forward_mode_refusals(on_host, data):
    pos, inv, q, k, tq, _ = data
    with fwd.dual_level():
        dual = fwd.make_dual(q, tq)
        with pytest.raises(ValueError, match="gradients through out"):
            rotary.rotate_positions(dual, k, pos, inv, SECTIONS, out=(torch.empty_like(q), torch.empty_like(k)))
        with pytest.raises(ValueError, match="no gradient"):
            rotary.rotate_positions(q, k, pos, inv, SECTIONS, out=(fwd.make_dual(torch.empty_like(q), tq), torch.empty_like(k)))
        with pytest.raises(ValueError, match="inv_freq"):
            rotary.rotate_positions(q, k, pos, fwd.make_dual(inv, torch.ones_like(inv)), SECTIONS)


def test_reverse_mode(on_host, data):
    pos, inv, q, k, wq, wk = data
    a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
    y, z = rotary.rotate_positions(a, b, pos, inv, SECTIONS)
    dq, dk = torch.autograd.grad((y, z), (a, b), (wq, wk))
    assert torch.equal(dq, turn(wq, pos, inv, True)) and torch.equal(dk, turn(wk, pos, inv, True))
