"""The sequence operators at the calls that are easily got wrong: closed gates, long memories, narrow types, odd strides, repeated calls."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def normal(gpu, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return lambda *s, k=1.0, dtype=torch.float32: (torch.randn(*s, generator=g, device=gpu) * k).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,F", [(3996, 1000, 512), (300, 72, 4100), (4, 1024, 4096)])
def test_ff_same_bits_between_other_calls_and_how_far_from_64(gpu, dtype, M, K, F):
    """A pass gives the same bits at every call, other passes in between; and its 16-bit gradients are off by their own rounding and by that of dg and du, two
    independent errors of one size: sqrt 2 times the norm of the first alone (a twentieth for what both are sampled by)."""
    from videometamaterials_amd import gated_feed_forward
    n = normal(gpu, M)

    def inputs():
        return [n(M, K, dtype=dtype), *(n(F, K, k=K ** -0.5, dtype=dtype) for _ in range(2)), *(n(F, k=0.1, dtype=dtype) for _ in range(2))], n(M, F, dtype=dtype)

    def run(leaves, dh):
        leaves = [v.detach().requires_grad_() for v in leaves]
        h = gated_feed_forward(*leaves, activation="gelu")
        return (h.detach(), *torch.autograd.grad(h, leaves, dh))
    (one, dh), (other, dh2) = inputs(), inputs()
    want = run(one, dh)
    for _ in range(4):
        run(other, dh2)
        assert all(torch.equal(a, b) for a, b in zip(run(one, dh), want))
    if dtype == torch.float32:
        return
    x, wg, wu, bg, bu = (v.double() for v in one)
    lin = torch.nn.functional.linear
    g, u = lin(x, wg, bg), lin(x, wu, bu)
    p = torch.special.ndtr(g)
    dg, du = dh.double() * u * (p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)), dh.double() * g * p
    exact = (g * p * u, dg @ wg + du @ wu, dg.t().contiguous() @ x, du.t().contiguous() @ x)
    for k, (got, w) in enumerate(zip(want, exact)):
        off, alone = float((got.double() - w).norm()), float((w.to(dtype).double() - w).norm())
        assert off < (1.05 if k == 0 else 1.05 * math.sqrt(2)) * alone, k


def scan_reference(x, gate, h0, dy, dlast):
    """y, last, dx, dgate, dh0 of the recurrence in 64 bits, and beside each the same sums over absolute values, by which its error is measured: an operator that keeps
    every factor to a few roundings of fp32 stays within those roundings of them, however small a result is."""
    x, gate, h0, dy, dlast = (v.detach().double().cpu() for v in (x, gate, h0, dy, dlast))
    L = x.shape[1]
    f, i = torch.sigmoid(gate), torch.sigmoid(-gate)

    def run(x, h0, dy, dlast, less):
        h, before, y = h0, [], []
        for t in range(L):
            before.append(h)
            h = f[:, t] * h + i[:, t] * x[:, t]
            y.append(h)
        c, dx, dg = dlast, [None] * L, [None] * L
        for t in reversed(range(L)):
            dh = dy[:, t] + c
            dx[t], dg[t] = dh * i[:, t], dh * less(before[t], x[:, t]) * f[:, t] * i[:, t]
            c = f[:, t] * dh
        return torch.stack(y, 1), h, torch.stack(dx, 1), torch.stack(dg, 1), c
    return zip(run(x, h0, dy, dlast, lambda a, b: a - b), run(x.abs(), h0.abs(), dy.abs(), dlast.abs(), lambda a, b: a + b))


def scan_all(x, gate, h0, dy, dlast):
    from videometamaterials_amd import gated_linear_scan
    leaves = [v.detach().requires_grad_() for v in (x, gate, h0)]
    y, last = gated_linear_scan(*leaves)
    return (y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dy, dlast)))


def within(got, want, bound, what):
    off = (got.detach().double().cpu() - want).abs() - bound
    at = int(off.argmax())
    assert float(off.max()) <= 0, f"{what}: {float(got.flatten()[at])} for {float(want.flatten()[at])}, {float(bound.flatten()[at])} allowed, at {at}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 40, 300])
@pytest.mark.parametrize("x_size", [1.0, 0.0])
def test_scan_closed_gates(gpu, dtype, L, x_size):
    """Forget gates of e^-8 to e^-19 (and open ones beside them): dgate, dh0 and states that come through a closed gate are proportional to it, so it has to be
    right relative to itself.  A gate is off by (|g| + 4) U of itself; a state passes at most some 20 gates that are not closed before it is gone."""
    n = normal(gpu, 17)
    x, h0, dy, dlast = n(2, L, 24, k=x_size, dtype=dtype), n(2, 24), n(2, L, 24, dtype=dtype), n(2, 24)
    gate = torch.linspace(-19.0, -8.0, 24, device=gpu).expand(2, L, 24) + n(2, L, 24, k=0.3)
    gate[:, ::7, ::5] = 2.0
    gate = gate.to(dtype)
    rel = 8 * (float(gate.abs().max()) + 4) * U
    # What ends below a type's smallest normal number is a multiple of its smallest number (2^-24, 2^-133, 2^-149) and loses half of that, whatever its size: y, dx and
    # dgate once in their type, a state of fp32 at every gate it passes -- 1 / (1 - f) = 8.4 of them are alive behind open gates of f = sigmoid(2), twice that
    # for maps that were joined before they were applied.
    sub = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    small = 17 * 2.0 ** -150
    for what, got, (want, size) in zip(("y", "last", "dx", "dgate", "dh0"), scan_all(x, gate, h0, dy, dlast), scan_reference(x, gate, h0, dy, dlast)):
        held = (half_step(dtype) * want.abs() + sub) if got.dtype == dtype else 0.0
        within(got, want, held + (rel * size + small) * (1 + half_step(dtype)), what)


@pytest.mark.parametrize("kind", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32, torch.uint64])
def test_scan_lengths_of_every_integer_type(gpu, kind):
    """Sequences longer than the type can say, values outside 0 .. L."""
    from videometamaterials_amd import gated_linear_scan
    n = normal(gpu, 1)
    x, gate = n(4, 300, 8), n(4, 300, 8)
    info = torch.iinfo(kind)
    values = [info.min, info.max, 0, 77]
    y, last = gated_linear_scan(x, gate, lengths=torch.tensor(values, dtype=kind).to(gpu))
    want, _ = gated_linear_scan(x, gate)
    for b, v in enumerate(values):
        v = min(max(v, 0), 300)
        assert torch.equal(y[b, :v], want[b, :v]) and not y[b, v:].any()
        # (The last state of a padded sequence comes through maps that are joined in an order of L, not of v: another order of the same sums.  A step rounds three
        # times; a state is a mean of inputs that forgets by f <= sigmoid(4.5) a step, 1 / (1 - f) < 92 steps in all; twice, for the two orders.)
        alone = gated_linear_scan(x[b:b + 1, :v], gate[b:b + 1, :v])[1][0]
        assert float(gate.max()) < 4.5 and float((last[b] - alone).abs().max()) <= 2 * 3 * 92 * U * float(x.abs().max())
    with pytest.raises(ValueError):
        gated_linear_scan(x, gate, lengths=torch.ones(4, device=gpu, dtype=torch.bool))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_of_dimensions_of_one(gpu, dtype):
    """One token, one row, one channel: the stride of such a dimension says nothing, and may be any number in a tensor that counts as contiguous."""
    from videometamaterials_amd import gated_feed_forward
    n = normal(gpu, 3)
    far = (1 << 40) + 3

    def odd(t):
        return torch.as_strided(t, t.shape, [far if size == 1 else stride for size, stride in zip(t.shape, t.stride())])
    for B, L, D in ((3, 1, 64), (1, 1, 5), (1, 90, 20), (2, 90, 1), (1, 1, 1)):
        x, gate, dy = (n(B, L, D, dtype=dtype) for _ in range(3))
        h0, dlast = n(B, D), n(B, D)
        got, want = scan_all(odd(x), odd(gate), odd(h0), odd(dy), odd(dlast)), scan_all(x, gate, h0, dy, dlast)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (B, L, D)
    for M, K, F in ((1, 64, 24), (1, 1, 1), (5, 1, 3), (5, 8, 1), (1, 9, 7)):
        x, w, v, dh = n(M, K, dtype=dtype), n(F, K, dtype=dtype), n(F, K, dtype=dtype), n(M, F, dtype=dtype)
        out = []
        for change in (odd, lambda t: t):
            leaves = [change(t).requires_grad_() for t in (x, w, v)]
            h = gated_feed_forward(*leaves)
            out.append((h, *torch.autograd.grad(h, leaves, change(dh))))
        assert all(torch.equal(a, b) for a, b in zip(*out)), (M, K, F)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,F", [(7, 9), (8, 16), (40, 300)])
def test_ff_backward_without_rows_reads_nothing(gpu, dtype, K, F):
    """Through the C ABI: no rows, none of the inputs there, and the gradients of the weights are zero."""
    import ctypes as C
    from videometamaterials_amd import _native as N
    lib = N.lib()
    dw, db = torch.full((2, F, K), 7.0, device=gpu, dtype=dtype), torch.full((2, F), 7.0, device=gpu, dtype=dtype)
    d = N.GatedFFDesc(ldx=K, lddh=F, lddx=K, dw_gate=dw[0].data_ptr(), dw_up=dw[1].data_ptr(), db_gate=db[0].data_ptr(), db_up=db[1].data_ptr(), M=0, K=K, F=F,
                      type=TYPES.index(dtype))
    d.workspace_bytes = lib.vmm_gated_ff_workspace(C.byref(d), 1)
    room = torch.empty(max(d.workspace_bytes, 16), dtype=torch.uint8, device=gpu)
    d.workspace = room.data_ptr()
    N.check(lib.vmm_gated_ff_bwd(C.byref(d), torch.cuda.current_stream().cuda_stream), "backward")
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()


def test_smallest_bound_clips(gpu):
    """The smallest positive float32 is a bound like any other: values that it leaves are below it."""
    from videometamaterials_amd import clip_grad_norm_
    g = normal(gpu, 4)(5000)
    norm = clip_grad_norm_([g], 2.0 ** -149)
    assert float(norm) > 60 and not g.any()


def test_captured_backward_beside_an_eager_graph_of_the_same_leaves(gpu):
    """Refused while the eager graph lives; captured and replayed once it is gone."""
    from videometamaterials_amd import gated_feed_forward, gated_linear_scan
    from videometamaterials_amd._native import NativeError
    n = normal(gpu, 5)
    x, gate, w, v = n(2, 70, 16), n(2, 70, 16), n(24, 16), n(24, 16)
    leaves = [t.requires_grad_() for t in (x, gate, w, v)]
    dy = n(2, 70, 16)
    dh = n(2, 70, 24)
    scan = lambda: torch.autograd.grad(gated_linear_scan(x, gate)[0], (x, gate), dy)  # noqa: E731
    product = lambda: torch.autograd.grad(gated_feed_forward(x, w, v), (x, w, v), dh)  # noqa: E731
    side, scratch = torch.cuda.Stream(gpu), torch.zeros(4, device=gpu)
    behind = lambda: torch.autograd.grad(gated_linear_scan(2 * x[:, ::1], gate.detach())[0], (x,), dy)  # noqa: E731  (torch's own operations in between)
    for run, forward in ((scan, lambda: gated_linear_scan(x, gate)[0]), (product, lambda: gated_feed_forward(x, w, v)),
                         (behind, lambda: gated_linear_scan(x, gate.detach())[0])):
        alive = forward()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scratch.add_(1.0)
            with pytest.raises((NativeError, RuntimeError), match="eager graph"):
                run()
        want = torch.autograd.grad(alive, [t for t in leaves if t is not None], torch.ones_like(alive), allow_unused=True)
        assert any(d is not None and bool(torch.isfinite(d).all()) for d in want)
        del alive, want
        if run is product:  # what an eager graph holds and nobody asks a gradient of does not matter
            alive = gated_feed_forward(x.detach(), w, v.detach())
            run = lambda: torch.autograd.grad(gated_feed_forward(x, w, v), (x, v), dh)  # noqa: E731
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        for seed in range(3):
            with torch.no_grad():
                for t in leaves:
                    t.copy_(normal(gpu, 50 + seed)(*t.shape))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, run()))
            torch.cuda.synchronize()


def test_ff_products_of_fp32_values(gpu):
    """Single products (K = 1) of values whose parts are as large as parts get.  With wg = 64 the gate's pre-activation is 64 x without an error and silu passes it, so
    h = 64 x (x wu): the product's parts that are left out are 2^-24 = U of it at most, the product with 64 x rounds by U.  The last sum adds the largest product to
    a smaller accumulator, which the matrix unit then floors to the sum's last place (1 * 1 + 1.5 2^-24 gives 1, 1 * 1 - 2^-30 gives 1 - 2^-24; an accumulator
    that is the larger is rounded to nearest): up to 2 U, always downwards; the sums before it lose 2^-7 of that each.
    What is left out has no side, so the mean over 2^18 products is that of the floor alone, half a last place: between zero and -U (parts that are cut would add
    0.63 U to it)."""
    from videometamaterials_amd import gated_feed_forward
    bits = torch.randint(0, 1 << 23, (4096,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    bits[:8] = torch.tensor([0x00ffff, 0x7fffff, 0x007fff, 0x008000, 0x7f7fff, 0x00ff7f, 0x7e8080, 0x7fff80])
    value = (bits | 0x3f800000).view(torch.float32)
    x, wu = value[:, None].to(gpu), value[:64, None].contiguous().to(gpu)
    h = gated_feed_forward(x, torch.full_like(wu, 64.0), wu).double().cpu()
    want = 64 * value.double()[:, None] ** 2 * value[:64].double()
    off = (h - want) / want
    assert float(off.abs().max()) <= (1 + 2 + 1 + 2.0 ** -5) * U
    assert -1.05 * U < float(off.mean()) < 0.05 * U
    # next to the largest value a part is not rounded up to infinity; an infinite operand gives NaN
    top = torch.tensor([[torch.finfo(torch.float32).max], [-3.39e38], [float("inf")], [1.0]], device=gpu)
    one = torch.tensor([[0.25]], device=gpu)
    h = gated_feed_forward(top, torch.zeros_like(one), one)
    assert not h[:2].any() and bool(torch.isnan(h[2]).all()) and not h[3].any()


def recurrence(f, b, h):
    """h_t = f_t h_(t-1) + b_t over dimension 1 in 64 bits, in pieces that are walked side by side and then joined."""
    B, L, D = f.shape
    c = max(1, math.isqrt(L))
    n = -(-L // c)
    pad = n * c - L
    f = torch.cat([f, torch.ones(B, pad, D, dtype=f.dtype)], 1).view(B, n, c, D)
    b = torch.cat([b, torch.zeros(B, pad, D, dtype=b.dtype)], 1).view(B, n, c, D)
    out, through = torch.empty_like(b), torch.empty_like(f)
    p, q = torch.ones_like(f[:, :, 0]), torch.zeros_like(b[:, :, 0])
    for t in range(c):
        p, q = p * f[:, :, t], q * f[:, :, t] + b[:, :, t]
        through[:, :, t], out[:, :, t] = p, q
    for k in range(n):
        out[:, k] += through[:, k] * h[:, None]
        h = out[:, k, -1]
    return out.view(B, n * c, D)[:, :L]


def scan_with_bounds(x, gate, h0, dy, dlast):
    """(name, value in 64 bits, sum of absolute values, bound) of y, last, dx, dgate, dh0.  The bound follows the decay of each channel: a gate that is open (f > i) is off by its
    own rounding and by i / f times the (|g| + 6) U of i, a closed one by (|g| + 6) U, and a step rounds three times more (sum and map); a state's error is what the step before
    hands on, E_t = f (E_(t-1) + 2 (rho + 3 U) H_(t-1)) + 2 (|g| + 8) U i |x|, with H the same recurrence of absolute values, and a factor of two for how maps are joined."""
    x, g, h0, dy, dlast = (v.detach().double().cpu() for v in (x, gate, h0, dy, dlast))
    f, i = torch.sigmoid(g), torch.sigmoid(-g)
    rho, wide = 2 * U * (4 + torch.clamp(i / f, max=1.0) * (g.abs() + 6)), 2 * U * (g.abs() + 8)

    def shifted(first, rest):
        return torch.cat([first[:, None], rest[:, :-1]], 1)
    h, H = recurrence(f, i * x, h0), recurrence(f, i * x.abs(), h0.abs())
    E = recurrence(f, f * rho * shifted(h0.abs(), H) + wide * i * x.abs(), torch.zeros_like(h0))
    before, Hb, Eb = shifted(h0, h), shifted(h0.abs(), H), shifted(torch.zeros_like(h0), E)

    def back(b, c):  # c_t = f_t (b_t + c_(t+1)), from the end
        return recurrence(f.flip(1), (f * b).flip(1), c).flip(1)

    def after(c, last):  # what step t gets from behind it
        return torch.cat([c[:, 1:], last[:, None]], 1)
    c, C = back(dy, dlast), back(dy.abs(), dlast.abs())
    dh, DH = dy + after(c, dlast), dy.abs() + after(C, dlast.abs())
    Ec = recurrence(f.flip(1), (f * rho * DH).flip(1), torch.zeros_like(h0)).flip(1)
    Ed = after(Ec, torch.zeros_like(h0)) + U * DH
    yield "y", h, H, E
    yield "last", h[:, -1], H[:, -1], E[:, -1]
    yield "dx", dh * i, DH * i, i * (Ed + wide * DH)
    yield "dgate", dh * (before - x) * f * i, DH * (Hb + x.abs()) * f * i, f * i * (Ed * (Hb + x.abs()) + DH * Eb + 2 * wide * DH * (Hb + x.abs()))
    yield "dh0", c[:, 0], C[:, 0], Ec[:, 0]


LONG = [(1, 800_000, 6), (1, 530_000, 4), (2, 20_011, 36), (2, 4_093, 101)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,D", LONG)
def test_scan_long_memories(gpu, dtype, B, L, D):
    """Sequences of thousands of steps and of more than 256 groups of 1024 (anchors), with memories of two steps to a million side by side: every output element by element,
    and the same calls in pieces of an eighth (fewer than 256 groups, whole ones), the state handed on.  A piece has the same maps, joined in another order: a state differs by
    one rounding for each of 16 units, 16 rows and 256 groups it comes through, twice."""
    n = normal(gpu, L)
    # a memory of e^lean steps; the state in front and its gradient are as large as what comes on the way
    lean = torch.linspace(0.0, 14.0, D, device=gpu)[torch.randperm(D, generator=torch.Generator().manual_seed(D)).to(gpu)]
    x, gate, h0 = n(B, L, D, dtype=dtype), (n(B, L, D, k=0.5) + lean).to(dtype), n(B, D)
    dy, dlast = n(B, L, D, k=2e-3, dtype=dtype), n(B, D)
    got = scan_all(x, gate, h0, dy, dlast)
    sub = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    sizes = {}
    for value, (what, want, size, bound) in zip(got, scan_with_bounds(x, gate, h0, dy, dlast)):
        if value.dtype == dtype:
            bound = bound * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + sub
        within(value, want, bound + 17 * 2.0 ** -150, what)
        sizes[what] = size, want
    from videometamaterials_amd import gated_linear_scan
    leaves = [v.detach().requires_grad_() for v in (x, gate, h0)]
    h, ys, piece = leaves[2], [], -(-L // 8 // 1024) * 1024
    for t in range(0, L, piece):
        y, h = gated_linear_scan(leaves[0][:, t:t + piece], leaves[1][:, t:t + piece], h)
        ys.append(y)
    pieces = (torch.cat(ys, 1).detach(), h.detach(), *torch.autograd.grad((torch.cat(ys, 1), h), leaves, (dy, dlast)))
    joins = 2 * (16 + 16 + 256) * U
    channel = lambda v: v.reshape(-1, D).norm(dim=0)  # noqa: E731
    for value, other, (what, (size, want)) in zip(got, pieces, sizes.items()):
        step = 2 * half_step(dtype) if value.dtype == dtype else 0.0
        within(value, other.double().cpu(), 2 * joins * size + step * other.double().cpu().abs() + 2 * sub, what + " in pieces")
        if value.dim() == 3:  # (this bound is small beside the results, in the longest memories too: an output of zeros would not pass)
            assert bool((channel(2 * joins * size) < 0.2 * channel(want)).all()), (what, channel(2 * joins * size) / channel(want))


def test_gradients_that_are_lazily_negated(gpu):
    """The imaginary part of a conjugated tensor is its negative in memory, whatever its strides."""
    from videometamaterials_amd import gated_feed_forward, gated_linear_scan
    n = normal(gpu, 9)

    def negated(*shape):
        t = torch.complex(n(*shape), n(*shape)).conj().imag
        assert t.is_neg()
        return t
    for B, L, D in ((2, 70, 1), (1, 1, 1), (2, 70, 12)):
        x, gate = n(B, L, D).requires_grad_(), n(B, L, D).requires_grad_()
        y, last = gated_linear_scan(x, gate)
        dy, dlast = negated(B, L, D), negated(B, D)
        got = torch.autograd.grad((y, last), (x, gate), (dy, dlast), retain_graph=True)
        want = torch.autograd.grad((y, last), (x, gate), (dy.resolve_neg().contiguous(), dlast.resolve_neg().contiguous()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        w, v = n(D, D).requires_grad_(), n(D, D)
        h = gated_feed_forward(x, w, v)
        dh = negated(B, L, D)
        got = torch.autograd.grad(h, (x, w), dh, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(h, (x, w), dh.resolve_neg().contiguous())))


def test_ff_range_of_fp32_operands(gpu):
    """Powers of two on the other side show an operand as it is taken: exactly from 2^-110 up to the largest, and below rounded to a multiple of 2^-133."""
    from videometamaterials_amd import gated_feed_forward
    unit = torch.rand(500, generator=torch.Generator().manual_seed(2), dtype=torch.float64) + 1
    gate = torch.tensor([[0.0, 64.0]], device=gpu)
    for e in (127, 120, 40, 0, -60, -109, -110, -111, -118, -126, -131):
        v = (unit * 2.0 ** e).clamp(max=torch.finfo(torch.float32).max).float()
        other = 2.0 ** max(-100, min(100, -e))
        two = torch.stack([v, torch.ones_like(v)], 1).to(gpu)
        got = gated_feed_forward(two, gate, torch.tensor([[other, 0.0]], device=gpu)).double().cpu()[:, 0] / 64 / other
        as_weight = gated_feed_forward(torch.tensor([[other, 1.0]], device=gpu), gate.expand(500, 2).contiguous(), (two * torch.tensor([1.0, 0.0], device=gpu))).double().cpu()[0] / 64 / other
        assert torch.equal(got, as_weight)
        if e >= -110:
            assert torch.equal(got, v.double()), e
        else:
            assert float((got - v.double()).abs().max()) <= 2.0 ** -134, e


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [50, 200, 3000])
def test_scan_gradients_of_extreme_gates(gpu, dtype, L):
    """Gates of 200, infinity and the type's largest value, both signs: all or nothing, and no gradient of their own.  A NaN gate reaches what comes behind it forwards and what
    lies before it backwards, and nothing else."""
    n = normal(gpu, 12)
    x, gate, h0, dy, dlast = n(1, L, 8, dtype=dtype), n(1, L, 8, dtype=dtype), n(1, 8), n(1, L, 8, dtype=dtype), n(1, 8)
    top = torch.finfo(dtype).max
    for d, g in enumerate((200.0, -200.0, math.inf, -math.inf, top, -top)):
        gate[..., d] = g
    at = L // 2
    gate[0, at, 7] = math.nan
    y, last, dx, dgate, dh0 = (v.double().cpu() for v in scan_all(x, gate, h0, dy, dlast))
    h, dh, dl = h0.double().cpu()[0], dy.double().cpu()[0], dlast.double().cpu()[0]
    for d in (0, 2, 4):  # the state stands: its gradient is the sum of all that is asked of it, 64 bits of which the sum of L rounded steps knows (L + 8) U
        assert torch.equal(y[0, :, d], h[d].float().to(dtype).double().expand(L)) and not dx[0, :, d].any() and not dgate[0, :, d].any()
        assert abs(float(dh0[0, d] - dh[:, d].sum() - dl[d])) <= (L + 8) * U * float(dh[:, d].abs().sum() + dl[d].abs())
    for d in (1, 3, 5):  # every step is its own input
        assert torch.equal(y[0, :, d], x.double().cpu()[0, :, d]) and not dgate[0, :, d].any() and float(dh0[0, d]) == 0.0
        assert torch.equal(dx[0, :-1, d], dh[:-1, d]) and torch.equal(dx[0, -1, d], (dh[-1, d] + dl[d]).float().to(dtype).double())
    assert bool(torch.isfinite(y[0, :at, 7]).all()) and bool(torch.isnan(y[0, at:, 7]).all()) and bool(torch.isnan(last[0, 7]))
    assert bool(torch.isnan(dx[0, :at, 7]).all()) and bool(torch.isfinite(dx[0, at + 1:, 7]).all()) and bool(torch.isnan(dh0[0, 7]))
    assert all(bool(torch.isfinite(v[..., 6]).all()) for v in (y, last, dx, dgate, dh0))
