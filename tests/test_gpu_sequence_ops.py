"""The gated linear scan, the gated feed-forward product and the clipped optimizer against plain 64-bit implementations; tolerances follow from the arithmetic
and are stated where they are formed."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32, relative


def half_step(t):
    return torch.finfo(t).eps / 2


def close(got, want, bound, what):
    """|got - want| <= bound elementwise, and no NaN where none is wanted."""
    got, want, bound = got.double().cpu(), want.double().cpu(), torch.as_tensor(bound, dtype=torch.float64).cpu()
    off = (got - want).abs() - bound
    assert got.shape == want.shape and bool(torch.isfinite(got).all()) and float(off.max() if off.numel() else 0.0) <= 0.0, \
        f"{what}: {float((got - want).abs().max()):.3e} off, {float(off.max()):.3e} over the bound"


# ---------------------------------------------------------------- the scan


def scan_reference(x, gate, h0, lengths, dy=None, dlast=None):
    """Step by step in 64 bits on the CPU: (y, last[, dx, dgate, dh0]), and the size that each gradient's sums reach in absolute values."""
    x, g = x.detach().double().cpu(), gate.detach().double().cpu()
    B, L, D = x.shape
    h = torch.zeros(B, D, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    lens = torch.full((B,), L) if lengths is None else lengths.cpu().long().clamp(0, L)
    live = torch.arange(L)[None, :] < lens[:, None]
    f, i = torch.sigmoid(g), torch.sigmoid(-g)
    ys, before = torch.zeros(B, L, D, dtype=torch.float64), torch.zeros(B, L, D, dtype=torch.float64)
    for t in range(L):
        before[:, t] = h
        m = live[:, t, None]
        h = torch.where(m, f[:, t] * h + i[:, t] * torch.where(m, x[:, t], 0.0), h)
        ys[:, t] = torch.where(m, h, 0.0)
    if dy is None:
        return ys, h
    dy, c = dy.detach().double().cpu(), dlast.detach().double().cpu()
    size = c.abs()
    dx, dg, sizes = torch.zeros_like(ys), torch.zeros_like(ys), torch.zeros_like(ys)
    for t in reversed(range(L)):
        m = live[:, t, None]
        dh, sz = torch.where(m, dy[:, t], 0.0) + c, torch.where(m, dy[:, t].abs(), 0.0) + size
        dx[:, t] = torch.where(m, dh * i[:, t], 0.0)
        dg[:, t] = torch.where(m, dh * (before[:, t] - x[:, t]) * f[:, t] * i[:, t], 0.0)
        sizes[:, t] = sz
        c, size = torch.where(m, f[:, t] * dh, c), torch.where(m, f[:, t] * sz, size)
    return ys, h, dx, dg, c, sizes


def scan_bounds(x, gate, h0, L):
    """Relative error per step: exp2's argument, |g| U (what is left of it in fp32: less), and some eight roundings (exp2, rcp, sums and products, the maps'
    composition), each U; a state is an average of inputs, so a step adds that much of the largest, and no more than L steps do."""
    big = max(float(x.abs().max()), float(h0.abs().max()) if h0 is not None else 0.0)
    per_step = (float(gate.detach().float().abs().clamp(max=104).max()) + 8) * U
    return big, per_step * (L + 4)


def scan_inputs(gpu, dtype, B, L, D, joined, state, seed=0, lean=6.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    both = torch.randn(B, L, 2 * D, generator=g, device=gpu)
    both[..., D:] += torch.linspace(-1.0, lean, D, device=gpu)
    both = both.to(dtype)
    x, gate = (both[..., :D], both[..., D:]) if joined else (both[..., :D].contiguous(), both[..., D:].contiguous())
    h0 = torch.randn(B, D, generator=g, device=gpu) if state else None
    return x.detach(), gate.detach(), h0, torch.randn(B, L, D, generator=g, device=gpu).to(dtype), torch.randn(B, D, generator=g, device=gpu)


def check_scan(x, gate, h0, lengths, dy, dlast):
    from videometamaterials_amd import gated_linear_scan
    leaves = [x.requires_grad_(), gate.requires_grad_()] + ([h0.requires_grad_()] if h0 is not None else [])
    y, last = gated_linear_scan(x, gate, h0, lengths)
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    want = scan_reference(x, gate, h0, lengths, dy, dlast)
    L, t = x.shape[1], x.dtype
    big, rel = scan_bounds(x, gate, h0, L)
    sub = 2.0 ** -25 if t == torch.float16 else 0.0  # (half a step of the subnormal numbers)
    assert y.dtype == t and last.dtype == torch.float32 and grads[0].dtype == t
    close(y, want[0], half_step(t) * want[0].abs() + rel * big + sub, "y")
    close(last, want[1], U * want[1].abs() + rel * big, "last")
    close(grads[0], want[2], half_step(t) * want[2].abs() + rel * want[5] + sub, "dx")
    close(grads[1], want[3], half_step(t) * want[3].abs() + 3 * rel * want[5] * big + sub, "dgate")  # (h - x is up to twice the largest, f i a quarter)
    if h0 is not None:
        close(grads[2], want[4], U * want[4].abs() + rel * (want[5][:, 0] if L else dlast.abs().cpu()), "dh0")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,D,joined,state,ragged", [
    (1, 1, 1, False, True, False), (3, 1, 5, True, False, False), (2, 2, 64, True, True, False), (2, 63, 65, False, False, False), (2, 64, 68, True, True, False),
    (2, 65, 130, True, False, True), (1, 128, 4, False, True, False), (3, 129, 33, True, True, True), (5, 200, 100, True, False, True), (2, 1023, 12, False, False, False),
    (2, 1024, 20, True, True, False), (1, 1025, 72, True, False, True), (33, 70, 9, False, True, True), (1, 2100, 3, False, True, False)])
def test_scan_against_steps(gpu, dtype, B, L, D, joined, state, ragged):
    x, gate, h0, dy, dlast = scan_inputs(gpu, dtype, B, L, D, joined, state)
    lengths = None
    if ragged:  # no step at all, one, all of them, and values outside 0 .. L
        lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
        lengths[:5] = torch.tensor([0, L + 7, 1, -3, L], dtype=torch.int32)[:B]
        lengths = lengths.to(gpu)
    check_scan(x, gate, h0, lengths, dy, dlast)


def test_scan_beyond_the_first_anchors(gpu):
    """More than 256 groups of 1024 steps: the states come from anchors."""
    L = 3 * 256 * 1024 + 77
    x, gate, h0, dy, dlast = scan_inputs(gpu, torch.float32, 1, L, 4, True, True, lean=12.0)
    from videometamaterials_amd import gated_linear_scan
    leaves = [x.requires_grad_(), gate.requires_grad_(), h0.requires_grad_()]
    dy = dy * 1e-3
    y, last = gated_linear_scan(x, gate, h0)
    dx, dg, dh0 = torch.autograd.grad((y, last), leaves, (dy, dlast))
    # 64 bits in pieces side by side, which are then joined
    f, b = torch.sigmoid(gate.detach().double()), torch.sigmoid(-gate.detach().double()) * x.detach().double()

    def walk(f, b, h):
        n, c = 1024, -(-f.shape[1] // 1024)
        pad = n * c - f.shape[1]
        ff = torch.cat([f, torch.ones(1, pad, 4, device=gpu, dtype=torch.float64)], 1).view(c, n, 4)
        bb = torch.cat([b, torch.zeros(1, pad, 4, device=gpu, dtype=torch.float64)], 1).view(c, n, 4)
        p, q, out, through = torch.ones_like(ff[:, 0]), torch.zeros_like(bb[:, 0]), torch.empty_like(bb), torch.empty_like(ff)
        for t in range(n):
            p, q = p * ff[:, t], q * ff[:, t] + bb[:, t]
            through[:, t], out[:, t] = p, q
        for k in range(c):
            out[k] += through[k] * h
            h = out[k, -1]
        return out.view(1, -1, 4)[:, :f.shape[1]]
    want = walk(f, b, h0.detach().double())
    memory = 1.0 / float(torch.sigmoid(-gate.detach().double()).min())  # no error outlives the longest memory
    big, rel = float(x.abs().max()), (float(gate.abs().max()) + 8) * U * memory
    rel = min(rel, 2e-3)
    close(y, want, U * want.abs() + rel * big, "y")
    close(last, want[:, -1], rel * big, "last")
    c = walk(f.flip(1), (f * dy.double()).flip(1), dlast.double()).flip(1)
    dh = dy.double() + torch.cat([c[:, 1:], dlast.double()[:, None]], 1)
    size = float(dh.abs().max())
    close(dx, dh * torch.sigmoid(-gate.detach().double()), 2 * rel * size, "dx")
    close(dh0, c[:, 0], 2 * rel * size, "dh0")


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_does_not_read_behind_a_length(gpu, dtype):
    """NaN and infinities behind the lengths reach nothing; what is live is bit for bit what it is without them."""
    from videometamaterials_amd import gated_linear_scan
    x, gate, h0, dy, dlast = scan_inputs(gpu, dtype, 4, 150, 24, True, True)
    lengths = torch.tensor([0, 1, 64, 149], device=gpu)
    out = []
    for bad in (0.0, float("nan"), float("inf"), torch.finfo(dtype).min):
        behind = (torch.arange(150, device=gpu)[None] >= lengths[:, None])[..., None]
        leaves = [torch.where(behind, torch.tensor(bad, dtype=dtype, device=gpu), v).requires_grad_() for v in (x, gate)] + [h0.clone().requires_grad_()]
        y, last = gated_linear_scan(*leaves, lengths=lengths)
        out.append((y, last) + torch.autograd.grad((y, last), leaves, (torch.where(behind, torch.tensor(bad, dtype=dtype, device=gpu), dy), dlast)))
        assert float(torch.where(behind, y, 0).abs().max()) == 0.0 and all(float(torch.where(behind, d, 0).abs().max()) == 0.0 for d in out[-1][2:4])
        assert torch.equal(last[0], h0[0])
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


def test_scan_extreme_gates(gpu):
    """Gates whose exponentials leave fp32: keep everything, take everything, NaN stays in its own channel."""
    from videometamaterials_amd import gated_linear_scan
    for dtype in TYPES:
        x = torch.randn(1, 100, 8, device=gpu).to(dtype)
        gate = torch.zeros_like(x)
        top = torch.finfo(dtype).max
        gate[..., 0], gate[..., 1], gate[..., 2], gate[..., 3] = 200.0, -200.0, float("inf"), -float("inf")
        gate[..., 4], gate[..., 5] = top, -top
        gate[0, 50, 6] = float("nan")
        h0 = torch.randn(1, 8, device=gpu)
        y, last = gated_linear_scan(x, gate, h0)
        for keep in (0, 2, 4):
            assert torch.equal(y[0, :, keep], h0[0, keep].to(dtype).expand(100)) and last[0, keep] == h0[0, keep]
        for take in (1, 3, 5):
            assert torch.allclose(y[..., take].float(), x[..., take].float(), rtol=1e-6, atol=0)
        assert bool(torch.isfinite(y[..., 7]).all()) and bool(torch.isfinite(y[0, :50, 6]).all()) and bool(torch.isnan(y[0, 50:, 6]).all())


def test_scan_layouts(gpu):
    """Time before batch, expanded inputs (whose gradients are sums), rows that start at odd places, neighbours that are not next to each other."""
    from videometamaterials_amd import gated_linear_scan
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.randn(90, 3, 20, generator=g, device=gpu).transpose(0, 1)
    gate = torch.randn(3, 20, 90, generator=g, device=gpu).transpose(1, 2)
    dy, dlast = torch.randn(3, 90, 20, generator=g, device=gpu).transpose(0, 1).contiguous().transpose(0, 1), torch.randn(20, 3, generator=g, device=gpu).t()
    check_scan(x.detach(), gate.detach(), None, None, dy, dlast)
    flat = torch.randn(1 + 3 * 90 * 41, generator=g, device=gpu).bfloat16()
    odd = flat[1:].view(3, 90, 41)
    check_scan(odd[..., :20].detach(), odd[..., 21:].detach(), None, None, dy.bfloat16(), dlast)
    one, h0 = torch.randn(1, 1, 20, generator=g, device=gpu, requires_grad=True), torch.randn(1, 20, generator=g, device=gpu, requires_grad=True)
    gate = gate.detach().contiguous()
    y, last = gated_linear_scan(one.expand(3, 90, 20), gate, h0.expand(3, 20))
    d1, dh = torch.autograd.grad((y, last), (one, h0), (dy, dlast))
    full, hfull = one.detach().expand(3, 90, 20).contiguous().requires_grad_(), h0.detach().expand(3, 20).contiguous().requires_grad_()
    y2, last2 = gated_linear_scan(full, gate, hfull)
    e1, eh = torch.autograd.grad((y2, last2), (full, hfull), (dy, dlast))
    assert torch.equal(y, y2) and torch.allclose(d1, e1.sum((0, 1), keepdim=True), rtol=1e-5, atol=1e-5) and torch.allclose(dh, eh.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)


def test_scan_one_token_at_a_time(gpu):
    """A sequence in calls of one step, the state handed on, is the sequence in one call (both are within the bound of the same sums)."""
    from videometamaterials_amd import gated_linear_scan
    x, gate, h0, _, _ = scan_inputs(gpu, torch.bfloat16, 3, 70, 40, True, True)
    with torch.no_grad():
        y, last = gated_linear_scan(x, gate, h0)
        h, steps = h0, []
        for t in range(70):
            yt, h = gated_linear_scan(x[:, t:t + 1], gate[:, t:t + 1], h)
            steps.append(yt)
    big, rel = scan_bounds(x, gate, h0, 70)
    close(h, last, 2 * rel * big, "state")
    close(torch.cat(steps, 1), y, 2 * rel * big + 2 * half_step(torch.bfloat16) * y.double().cpu().abs(), "y")


def test_scan_partial_gradients_and_empty_sequences(gpu):
    from videometamaterials_amd import gated_linear_scan
    x, gate, h0, dy, dlast = scan_inputs(gpu, torch.float32, 2, 100, 8, False, True)
    for v in (x, gate, h0):
        v.requires_grad_()
    y, last = gated_linear_scan(x, gate, h0)
    both = torch.autograd.grad((y, last), (x, gate, h0), (dy, dlast), retain_graph=True)
    from_y = torch.autograd.grad(y, (x, gate, h0), dy, retain_graph=True)
    from_last = torch.autograd.grad(last, (x, gate, h0), dlast, retain_graph=True)
    for a, b, c in zip(both, from_y, from_last):
        assert torch.allclose(a, b + c, rtol=1e-5, atol=1e-5)
    only = torch.autograd.grad(y, gate, dy)[0]
    assert torch.equal(only, from_y[1])
    empty = torch.zeros(2, 0, 8, device=gpu, requires_grad=True)
    y, last = gated_linear_scan(empty, empty, h0)
    assert y.shape == (2, 0, 8) and torch.equal(last, h0) and torch.equal(torch.autograd.grad(last, h0, dlast)[0], dlast)
    y, last = gated_linear_scan(empty.detach(), empty.detach())
    assert float(last.abs().max()) == 0.0
    y, last = gated_linear_scan(torch.zeros(0, 5, 8, device=gpu), torch.zeros(0, 5, 8, device=gpu))
    assert y.shape == (0, 5, 8) and last.shape == (0, 8)


def test_scan_gradients_against_differences(gpu):
    """Central differences of the operator itself, fp32, in random directions: with steps of 2^-6 the third-order term is below 2e-3 of the first for these sums
    (derivatives of sigmoid are at most 1), the rounding of a sum of 600 terms over the step below 1e-3."""
    from videometamaterials_amd import gated_linear_scan
    x, gate, h0, dy, dlast = scan_inputs(gpu, torch.float32, 2, 75, 4, False, True, lean=2.0)
    leaves = [v.requires_grad_() for v in (x, gate, h0)]

    def value(*v):
        with torch.no_grad():
            y, last = gated_linear_scan(*v)
            return float((y.double() * dy.double()).sum() + (last.double() * dlast.double()).sum())
    y, last = gated_linear_scan(*leaves)
    grads = torch.autograd.grad((y, last), leaves, (dy, dlast))
    g = torch.Generator(device=gpu).manual_seed(8)
    for k in range(3):
        for _ in range(3):
            d = torch.randn(leaves[k].shape, generator=g, device=gpu)
            step = 2.0 ** -6
            plus, minus = ([v.detach() + (sign * step * d if i == k else 0) for i, v in enumerate(leaves)] for sign in (1, -1))
            slope, size = float((grads[k].double() * d.double()).sum()), float((grads[k].double() * d.double()).abs().sum())
            assert abs((value(*plus) - value(*minus)) / (2 * step) - slope) < 3e-3 * size


# ---------------------------------------------------------------- the feed-forward product


def ff_reference(x, wg, wu, bg, bu, act, dh=None):
    """64 bits on the CPU, with the bound of each output: products of K terms lose (K + 8) U of their sum of absolute values (fp32 operands another 2^-22: the products
    of parts that are left out), the activation 2e-6 of its size, dg and du half a step of the type, results half a step."""
    t = x.dtype
    x, wg, wu = (v.detach().double().cpu() for v in (x, wg, wu))
    bg, bu = ((v.detach().double().cpu() if v is not None else 0.0) for v in (bg, bu))
    K, F = x.shape[1], wg.shape[0]
    unit = U + (2.0 ** -22 if t == torch.float32 else 0.0)
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    eg, eu = ((x.abs() @ w.abs().t()) * (K * U + 8 * unit) + 2 * U * v.abs() for w, v in ((wg, g), (wu, u)))
    if act == "silu":
        p = torch.sigmoid(g)
        a, slope = g * p, p * (1 + g * torch.sigmoid(-g))
    else:
        p = torch.special.ndtr(g)
        a, slope = g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    ea, es = 1.13 * eg + 2e-6 * g.abs(), 1.0 * eg + 2e-6 * (1 + g.abs())  # (slopes of both activations and of their derivatives)
    sub = 2.0 ** -25 if t == torch.float16 else 0.0
    half = half_step(t)
    out = [(a * u, half * (a * u).abs() + ea * u.abs() + a.abs() * eu + ea * eu + sub)]
    if dh is None:
        return out
    dh = dh.detach().double().cpu()
    dg, du = dh * u * slope, dh * a
    edg = half * dg.abs() + dh.abs() * (slope.abs() * eu + u.abs() * es + eu * es) + sub
    edu = half * du.abs() + dh.abs() * ea + sub
    M = x.shape[0]

    def product(*pairs):
        v = sum(p @ q for p, q, _ in pairs)
        n = sum(p.shape[1] for p, _, _ in pairs)
        e = sum(ep @ q.abs() + (p.abs() @ q.abs()) * (n * U + 8 * unit) for p, q, ep in pairs)
        return v, half * v.abs() + e + sub
    out.append(product((dg, wg, edg), (du, wu, edu)))
    out.append(product((dg.t(), x, edg.t())))
    out.append(product((du.t(), x, edu.t())))
    for d, e in ((dg, edg), (du, edu)):  # the sums are of the values before their rounding; bound as if after
        out.append((d.sum(0), half * d.sum(0).abs() + e.sum(0) + (M + 8) * U * d.abs().sum(0)))
    return out


def ff_inputs(gpu, dtype, M, K, F, bias, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    n = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=gpu) * k).to(dtype)  # noqa: E731
    return n(M, K), n(F, K, k=K ** -0.5), n(F, K, k=K ** -0.5), *((n(F, k=0.2), n(F, k=0.2)) if bias else (None, None)), n(M, F)


def check_ff(x, wg, wu, bg, bu, act, dh):
    from videometamaterials_amd import gated_feed_forward
    leaves = [v.requires_grad_() for v in (x, wg, wu, bg, bu) if v is not None]
    h = gated_feed_forward(x, wg, wu, bg, bu, activation=act)
    grads = torch.autograd.grad(h, leaves, dh)
    with torch.no_grad():
        assert torch.equal(h, gated_feed_forward(x, wg, wu, bg, bu, activation=act))  # the same products with and without gradients to come
    want = ff_reference(x, wg, wu, bg, bu, act, dh)
    for name, got, (w, e) in zip(("h", "dx", "dwg", "dwu", "dbg", "dbu"), (h,) + grads, want):
        assert got.dtype == x.dtype
        close(got, w, e, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,F,bias,act", [
    (1, 1, 1, True, "silu"), (1, 8, 8, False, "gelu"), (5, 3, 7, True, "silu"), (4, 64, 128, False, "silu"), (4, 1024, 260, True, "gelu"), (33, 65, 31, True, "gelu"),
    (129, 72, 130, True, "silu"), (300, 257, 65, False, "gelu"), (256, 64, 128, True, "silu"), (200, 520, 96, True, "silu"), (1000, 40, 52, False, "silu"),
    (700, 129, 1, True, "gelu"), (2, 2000, 9, False, "silu")])
def test_ff_against_products(gpu, dtype, M, K, F, bias, act):
    check_ff(*ff_inputs(gpu, dtype, M, K, F, bias)[:5], act, ff_inputs(gpu, dtype, M, K, F, bias)[5])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,F", [(4001, 24, 1600), (4001, 3200, 17), (24, 2561, 2560)])
def test_ff_large_tiles(gpu, dtype, M, K, F):
    """Sizes at which the forward, dx and the weight gradients take the large tiles, each with edges inside them and a short reduced length."""
    *args, dh = ff_inputs(gpu, dtype, M, K, F, True)
    check_ff(*args, "silu", dh)


def test_ff_layouts(gpu):
    """Leading dimensions, rows inside wider rows, expanded inputs, weights and gradients that are transposed views, starts at odd places."""
    from videometamaterials_amd import gated_feed_forward
    g = torch.Generator(device=gpu).manual_seed(2)
    for dtype in TYPES:
        wide = torch.randn(3, 50, 80, generator=g, device=gpu).to(dtype)
        wt, wu = torch.randn(40, 24, generator=g, device=gpu).to(dtype).t(), torch.randn(24, 41, generator=g, device=gpu).to(dtype)[:, 1:]
        plain = lambda v: v.contiguous()  # noqa: E731
        for x in (wide[..., 40:], wide[..., 3:43], wide[:1, :1, :40].expand(3, 50, 40), wide[..., :40].transpose(0, 1)):
            h = gated_feed_forward(x, wt, wu)
            assert h.shape == x.shape[:-1] + (24,) and torch.equal(h, gated_feed_forward(plain(x), plain(wt), plain(wu)))
    x, w, v, _, _, dh = ff_inputs(gpu, torch.float32, 60, 32, 48, False)
    x, w, v = x.requires_grad_(), w.requires_grad_(), v.requires_grad_()
    a = torch.autograd.grad(gated_feed_forward(x, w, v), (x, w, v), dh.t().contiguous().t())
    b = torch.autograd.grad(gated_feed_forward(x, w, v), (x, w, v), dh)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    s = torch.autograd.grad(gated_feed_forward(x, w, v).sum(), (x, w, v))  # (the gradient of a sum is an expanded one)
    t = torch.autograd.grad(gated_feed_forward(x, w, v), (x, w, v), torch.ones_like(dh))
    assert all(torch.equal(p, q) for p, q in zip(s, t))
    only = torch.autograd.grad(gated_feed_forward(x.detach(), w, v), v, dh)[0]
    assert torch.equal(only, b[2])
    assert gated_feed_forward(x.detach()[:0], w, v).shape == (0, 48)
    e = torch.autograd.grad(gated_feed_forward(x[:0], w, v).sum(), (x, w))
    assert all(float(d.abs().max()) == 0.0 for d in e)


def test_ff_gradients_against_differences(gpu):
    """Central differences in random directions, fp32: steps of 2^-5 along unit directions leave a third-order term far below 1e-3 of the sum's size."""
    from videometamaterials_amd import gated_feed_forward
    for act in ("silu", "gelu"):
        *leaves, dh = ff_inputs(gpu, torch.float32, 20, 12, 16, True, seed=4)
        leaves = [v.requires_grad_() for v in leaves]
        grads = torch.autograd.grad(gated_feed_forward(*leaves, activation=act), leaves, dh)
        g = torch.Generator(device=gpu).manual_seed(5)
        for k in range(5):
            d = torch.randn(leaves[k].shape, generator=g, device=gpu)
            d = d / d.norm()
            step = 2.0 ** -5
            with torch.no_grad():
                plus, minus = (float((gated_feed_forward(*[v + (s * step * d if i == k else 0) for i, v in enumerate(leaves)], activation=act).double() * dh.double()).sum())
                               for s in (1, -1))
            slope, size = float((grads[k].double() * d.double()).sum()), float((grads[k].double() * d.double()).abs().sum())
            assert abs((plus - minus) / (2 * step) - slope) < 2e-3 * size + 1e-3


def test_ff_extreme_activations(gpu):
    """Pre-activations far out, where the activation is zero or the identity, in each type."""
    from videometamaterials_amd import gated_feed_forward
    for dtype in TYPES:
        for act in ("silu", "gelu"):
            x = torch.tensor([[1.0], [-1.0]], device=gpu, dtype=dtype)
            wg = torch.tensor([0.0, 20.0, 150.0, 3e4], device=gpu, dtype=dtype)[:, None]
            h = gated_feed_forward(x, wg, torch.ones_like(wg), activation=act)
            want = x.float() * (torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu)(x.float() * wg.float().t())
            assert torch.allclose(h.float(), want, rtol=2 * half_step(dtype) + 1e-6, atol=1e-7)


# ---------------------------------------------------------------- norm, clipping, optimizer


def tensors(gpu, sizes, dtypes, scale=0.02, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=gpu) * scale).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


SIZES = [[1], [0, 5, 0], [4095, 4096, 4097, 1, 3], [100003], [7] * 400, [1 << 22, 17, 123457], list(range(1, 200))]


@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{max(s)}" for s in SIZES])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=["f32", "bf16", "f16", "mixed"])
def test_norm_and_clipping(gpu, sizes, dtypes):
    """The norm to the rounding of its fp32 result; clipped values to half a step of their type and three of fp32 (the bound, the factor, the product)."""
    from videometamaterials_amd import clip_grad_norm_, grad_norm
    gs = tensors(gpu, sizes, dtypes)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    got = grad_norm(gs)
    assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - want) <= 2 * U * want
    assert torch.equal(grad_norm(gs), got) and torch.equal(grad_norm(iter(gs)), got)
    before = [g.clone() for g in gs]
    assert torch.equal(clip_grad_norm_(gs, 2 * want + 1), got) and all(torch.equal(a, b) for a, b in zip(gs, before))  # within the bound: untouched
    versions = [g._version for g in gs]
    assert torch.equal(clip_grad_norm_(gs, want / 3), got)
    factor = want / 3 / (want + 1e-6)
    for g, b, v in zip(gs, before, versions):
        w = b.double() * factor
        close(g, w, (half_step(g.dtype) + 3 * U) * w.abs().cpu() + (2.0 ** -25 if g.dtype == torch.float16 else 0.0), "clipped")
        assert g._version > v
    if dtypes == [torch.float32]:
        ref = [b.clone().requires_grad_() for b in before]
        for r, b in zip(ref, before):
            r.grad = b.clone()
        torch.nn.utils.clip_grad_norm_(ref, want / 3)
        assert all(torch.allclose(g, r.grad, rtol=4e-6, atol=0) for g, r in zip(gs, ref))


def test_norm_of_large_tiny_and_infinite_values(gpu):
    from videometamaterials_amd import clip_grad_norm_, grad_norm
    for v in (3e38, 1e30, 1e-30, 1e-38):  # squares that fp32 does not hold
        t = torch.full((1000,), v, device=gpu)
        want = float(t[0]) * math.sqrt(1000)
        assert abs(float(grad_norm([t])) - want) <= 2 * U * want if want < 3.4e38 else torch.isinf(grad_norm([t]))
    for bad in (float("inf"), float("nan")):
        gs = [torch.ones(5000, device=gpu), torch.ones(10, device=gpu)]
        gs[1][3] = bad
        assert not torch.isfinite(grad_norm(gs))
        ref = [torch.ones(5000), torch.ones(10)]
        ref[1][3] = bad
        ps = [r.clone().requires_grad_() for r in ref]
        for p, r in zip(ps, ref):
            p.grad = r
        torch.nn.utils.clip_grad_norm_(ps, 1.0)
        clip_grad_norm_(gs, 1.0)
        assert all(torch.equal(torch.nan_to_num(g.cpu(), nan=7.0), torch.nan_to_num(p.grad, nan=7.0)) for g, p in zip(gs, ps))


def test_clipping_refuses_what_overlaps_and_views_with_gaps(gpu):
    from videometamaterials_amd import ClippedAdam, clip_grad_norm_, grad_norm
    a = torch.ones(100, device=gpu)
    assert abs(float(grad_norm([a, a])) - math.sqrt(200)) < 1e-5  # reading twice is no matter
    for pair in ([a, a], [a[:60], a[50:]], [a, a[99:]]):
        with pytest.raises(ValueError):
            clip_grad_norm_(pair, 1.0)
        assert torch.equal(a, torch.ones_like(a))
    clip_grad_norm_([a[50:], a[:50]], 1.0)  # neighbours, in any order
    assert abs(float(a.norm()) - 1.0) < 1e-5
    with pytest.raises(ValueError):
        grad_norm([a[::2]])
    with pytest.raises(ValueError):
        ClippedAdam([a, a]).step([torch.ones_like(a), torch.ones_like(a)])
    with pytest.raises(ValueError):
        ClippedAdam([a]).step([torch.ones(99, device=gpu)])
    with pytest.raises(ValueError):
        ClippedAdam([a]).step([])
    with pytest.raises(ValueError):
        ClippedAdam([a]).step([a])  # its own gradient


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_norm", [None, 1e9, 0.05])
def test_clipped_adam_against_the_formulas(gpu, dtype, max_norm):
    """Five steps against 64 bits.  Each step rounds m and v three times and p twice (6 U of their terms' sizes); sqrt, division and the factor are good to a few U,
    so an update is off by at most 16 U of itself and a weight by U of itself more."""
    from videometamaterials_amd import ClippedAdam
    sizes = [5, 4096, 8193, 1, 70001] + [11] * 100
    ps = tensors(gpu, sizes, [torch.float32], 0.1, 1)
    opt = ClippedAdam(ps, lr=1e-2, max_norm=max_norm)
    p64 = [p.double() for p in ps]
    m64, v64 = [torch.zeros_like(p) for p in p64], [torch.zeros_like(p) for p in p64]
    moved = [torch.zeros_like(p) for p in p64]
    for step in range(1, 6):
        gs = tensors(gpu, sizes, [dtype], 0.02, 10 + step)
        norm = opt.step(gs)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in gs))
        assert abs(float(norm) - want) <= 2 * U * want
        c = 1.0 if max_norm is None else min(1.0, max_norm / (want + 1e-6))
        for i, g in enumerate(gs):
            g = g.double() * c
            m64[i] = 0.9 * m64[i] + 0.1 * g
            v64[i] = 0.999 * v64[i] + 0.001 * g * g
            d = 1e-2 * (m64[i] / (1 - 0.9 ** step)) / ((v64[i] / (1 - 0.999 ** step)).sqrt() + 1e-8)
            p64[i] = p64[i] - d
            moved[i] += 1e-2  # (an update is at most about the step size; a small m, the difference of larger terms, keeps their error)
    for i, p in enumerate(ps):
        close(opt.exp_avgs[i], m64[i], 30 * U * 0.1 * c, "m")  # (|g| < 0.1)
        close(opt.exp_avg_sqs[i], v64[i], 60 * U * v64[i].cpu() + 1e-30, "v")
        big = moved[i].cpu() * (200 * U) + 5 * U * p64[i].abs().cpu()
        close(p, p64[i], big, "p")
    assert opt.steps_taken == 5


def test_clipped_adam_like_torch_and_missing_gradients(gpu):
    from videometamaterials_amd import ClippedAdam
    ps = [p.requires_grad_() for p in tensors(gpu, [300, 5000, 7], [torch.float32], 0.1)]
    qs = [p.detach().clone().requires_grad_() for p in ps]
    opt, ref = ClippedAdam(ps, lr=1e-3), torch.optim.Adam(qs, lr=1e-3)
    for step in range(4):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = tensors(gpu, [p.numel()], [torch.float32], 0.02, 50 + step * 3 + i)[0]
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
    assert all(torch.allclose(p, q, rtol=0, atol=3e-6) for p, q in zip(ps, qs))
    before = [p.detach().clone() for p in ps]
    moments = [m.clone() for m in opt.exp_avgs]
    ps[1].grad = None
    v = [p._version for p in ps]
    opt.step()
    assert torch.equal(ps[1], before[1]) and torch.equal(opt.exp_avgs[1], moments[1]) and not torch.equal(ps[0], before[0])
    assert ps[0]._version > v[0] and ps[1]._version == v[1]
    assert float(opt.step([None, None, None])) == 0.0
    ps[0].data = ps[0].data.clone()  # re-homed
    at = ps[0].detach().clone()
    opt.step()
    assert not torch.equal(ps[0], at)
    ps[0].data = torch.zeros(5, device=gpu)
    with pytest.raises(ValueError):
        opt.step([torch.zeros(300, device=gpu), None, None])


# ---------------------------------------------------------------- graphs, streams, the operators together


def everything(x, gate, h0, w, v, dy, dh):
    """Scan and feed-forward product of its states, with the gradients of both results."""
    from videometamaterials_amd import gated_feed_forward, gated_linear_scan
    leaves = [t.detach().requires_grad_() for t in (x, gate, h0, w, v)]
    y, last = gated_linear_scan(leaves[0], leaves[1], leaves[2])
    h = gated_feed_forward(y, leaves[3], leaves[4])
    return (y.detach(), last.detach(), h.detach()) + torch.autograd.grad((y, last, h), leaves, (dy, torch.ones_like(last), dh))


def layer_inputs(gpu, dtype, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    n = lambda *s, k=1.0: (torch.randn(*s, generator=g, device=gpu) * k).to(dtype)  # noqa: E731
    B, L, D, F = 3, 300, 64, 128
    return [n(B, L, D), n(B, L, D) + 2, torch.randn(B, D, generator=g, device=gpu), n(F, D, k=D ** -0.5), n(F, D, k=D ** -0.5), n(B, L, D), n(B, L, F)]


def test_operators_are_the_same_every_time_and_on_every_stream(gpu):
    a, b = layer_inputs(gpu, torch.bfloat16, 1), layer_inputs(gpu, torch.bfloat16, 2)
    ra, rb = everything(*a), everything(*b)
    side = [torch.cuda.Stream(gpu), torch.cuda.Stream(gpu)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):  # two streams at once
        for s, args in zip(side, (a, b)):
            with torch.cuda.stream(s):
                got.append(everything(*args))
    torch.cuda.synchronize()
    for k, r in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(r, (ra, rb)[k % 2]))


def test_captured_operators_replay(gpu):
    """Forward calls of all three kinds in two graphs, replayed in turn on new inputs with eager work between."""
    from videometamaterials_amd import clip_grad_norm_, gated_feed_forward, gated_linear_scan, grad_norm

    def calls(args, grads):
        with torch.no_grad():
            y, last = gated_linear_scan(args[0], args[1], args[2])
            h = gated_feed_forward(y, args[3], args[4])
            return y, last, h, grad_norm(grads), clip_grad_norm_(grads, 0.5)
    sets = []
    for seed in (1, 2):
        args, grads = layer_inputs(gpu, torch.float32, seed), tensors(gpu, [1000, 30000, 3], [torch.float32], 0.02, seed)
        s = torch.cuda.Stream(gpu)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            calls(args, [g.clone() for g in grads])
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls(args, grads)
        sets.append((args, grads, graph, out))
    for turn in range(4):
        for k, (args, grads, graph, out) in enumerate(sets):
            fresh = layer_inputs(gpu, torch.float32, 10 + 2 * turn + k)
            new = tensors(gpu, [1000, 30000, 3], [torch.float32], 0.02, 100 + turn)
            for a, f in zip(args, fresh):
                a.copy_(f)
            for g, f in zip(grads, new):
                g.copy_(f)
            graph.replay()
            want = calls(fresh, new)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, want)) and all(torch.equal(p, q) for p, q in zip(grads, new)), (turn, k)


def test_captured_training_pass_replays(gpu):
    """Forward and backward of the operators in one graph, replayed on new inputs with eager passes between, while an eager graph of the same tensors lives."""
    args = layer_inputs(gpu, torch.bfloat16, 7)
    from videometamaterials_amd import gated_linear_scan
    alive = gated_linear_scan(args[0].clone().requires_grad_(), args[1])
    s = torch.cuda.Stream(gpu)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        everything(*args)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = everything(*args)
    for turn in range(4):
        fresh = layer_inputs(gpu, torch.bfloat16, 20 + turn)
        for a, f in zip(args, fresh):
            a.copy_(f)
        graph.replay()
        want = everything(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), turn
    assert bool(torch.isfinite(alive[0]).all())


def test_gradients_are_differentiable_once_and_saved_tensors_are_watched(gpu):
    from videometamaterials_amd import gated_feed_forward, gated_linear_scan
    x, gate, w = (torch.randn(*s, device=gpu, requires_grad=True) for s in ((2, 70, 16), (2, 70, 16), (8, 16)))
    for value, leaf in ((lambda: gated_linear_scan(x, gate)[0], gate), (lambda: gated_feed_forward(x, w, w), w)):
        y = value()
        d = torch.autograd.grad(y, leaf, torch.ones_like(y), create_graph=True)[0]
        assert torch.equal(d.detach(), torch.autograd.grad(value(), leaf, torch.ones_like(y))[0])
        with pytest.raises(RuntimeError):
            d.sum().backward()
        y = value()
        with torch.no_grad():
            leaf.mul_(1.0)
        with pytest.raises(RuntimeError):
            y.sum().backward()


def test_clipped_adam_is_not_captured(gpu):
    from videometamaterials_amd import ClippedAdam
    p = torch.ones(100, device=gpu)
    opt, g, scratch = ClippedAdam([p]), torch.ones(100, device=gpu), torch.zeros(4, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scratch.add_(1.0)
        with pytest.raises(RuntimeError):
            opt.step([g])
    graph.replay()
    assert opt.steps_taken == 0 and float(p.sum()) == 100.0 and float(scratch[0]) == 1.0


def test_training_an_encoder_layer_with_all_of_them(gpu):
    """A layer of projection, scan and gated feed-forward, trained for some steps by the clipped optimizer, against the same layer of torch operations with
    clip_grad_norm_ and torch.optim.Adam: the weights stay together (both take the same ten steps of 1e-3; a step's relative error is that of its gradient)."""
    from videometamaterials_amd import ClippedAdam, gated_feed_forward, gated_linear_scan
    g = torch.Generator(device=gpu).manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    x, target = n(4, 51, 1), n(4, 51, 32)
    shapes = [(64, 1), (64,), (64, 32), (64, 32), (64,), (64,), (32, 64)]
    ps = [(n(*s) * 0.3).requires_grad_() for s in shapes]
    qs = [p.detach().clone().requires_grad_() for p in ps]

    def ours(p):
        z = x @ p[0].t() + p[1]
        y, _ = gated_linear_scan(z[..., :32], z[..., 32:])
        return ((y + gated_feed_forward(y, p[2], p[3], p[4], p[5]) @ p[6].t() - target) ** 2).mean()

    def plain(p):
        z = x @ p[0].t() + p[1]
        c, f = z[..., :32], torch.sigmoid(z[..., 32:])
        h, out = torch.zeros(4, 32, device=gpu), []
        for t in range(51):
            h = f[:, t] * h + (1 - f[:, t]) * c[:, t]
            out.append(h)
        y = torch.stack(out, 1)
        return ((y + (torch.nn.functional.silu(y @ p[2].t() + p[4]) * (y @ p[3].t() + p[5])) @ p[6].t() - target) ** 2).mean()
    opt, ref = ClippedAdam(ps, lr=1e-3, max_norm=0.1), torch.optim.Adam(qs, lr=1e-3)
    for _ in range(10):
        grads = torch.autograd.grad(ours(ps), ps)
        norm = opt.step(grads)
        ref.zero_grad()
        plain(qs).backward()
        want = torch.nn.utils.clip_grad_norm_(qs, 0.1)
        ref.step()
        assert abs(float(norm) - float(want)) < 1e-3 * float(want)
    for p, q in zip(ps, qs):
        assert float((p - q).abs().max()) < 1e-3  # a tenth of the way that ten steps can go
