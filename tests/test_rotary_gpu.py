"""Norm and rotation of query / key heads against the formulas in 64 bits.

Tolerances (u = 2^-24, half = half a step of the output's type, eps / 2):
* a sum of D products is added in at most n = 40 steps (8 per lane and 5 shuffles, or D / 32 and 5), so
  it is off by n u of the sum of absolute values, and 1/sqrt of the mean square by (n / 2 + 3) u;
* sine and cosine of an angle rounded to float32 inside [-pi, pi] are off by 2 u + 2 u;
* every output value adds at most 8 roundings.
Forward: half |y| + (n / 2 + 3 + 4 + 8) u (|n_a| + |n_b|), that is 40 u.  Backward: dot product and both
factors of 1/rms, 2 n + 20 = 100 u of r (|g| + |unit| mean |g unit|), with g by absolute terms."""
import pytest
import torch

import tiga as tg

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}   # steps of subnormals


def turn(x, angle, interleaved):
    pairs = angle.shape[-1]
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    y = x.clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def turn_magnitude(x, pairs, interleaved):
    x = x.abs()
    y = x.clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    y[..., a] = y[..., b] = x[..., a] + x[..., b]
    return y


def angles(positions, frequencies):
    f = frequencies.double() if frequencies.ndim == 2 else frequencies.double()[None]
    return positions.double().reshape(positions.shape[0], -1) @ f


def expected(x, w, angle, eps, interleaved):
    x = x.double()
    n = x if eps is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = n if w is None else n * w.double()
    return turn(n, angle, interleaved), turn_magnitude(n, angle.shape[-1], interleaved)


def assert_within(got, want, bound):
    excess = (got.double() - want).abs() - bound
    assert bool((excess <= 0).all()), f"worst excess {excess.max().item()} over a bound of {bound.max().item()}"


def make(tokens, heads, kv_heads, dim, pairs, axes, dtype, seed, limit=4000):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    packed = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=gen, device="cuda").to(dtype)
    q = packed[:, :heads * dim].view(tokens, heads, dim)
    k = packed[:, heads * dim:(heads + kv_heads) * dim].view(tokens, kv_heads, dim)
    positions = torch.randint(-limit, limit, (tokens, axes), generator=gen, device="cuda")
    frequencies = torch.rand(axes, pairs, generator=gen, device="cuda")
    if axes == 1:
        positions, frequencies = positions[:, 0].contiguous(), frequencies[0].contiguous()
    return q, k, positions, frequencies, gen


CASES = (
    # tokens, heads, kv_heads, dim, pairs, axes, interleaved, dtype
    (1, 1, 1, 2, 1, 1, False, torch.float32),
    (1, 32, 8, 128, 64, 1, False, torch.bfloat16),
    (7, 3, 1, 64, 32, 2, True, torch.float16),
    (5, 5, 5, 80, 20, 1, False, torch.bfloat16),         # half a rotation of 20 pairs: narrower pieces of a head
    (33, 4, 2, 96, 24, 3, False, torch.float16),
    (9, 2, 2, 96, 31, 1, True, torch.bfloat16),          # the turned values end inside a piece
    (9, 2, 2, 96, 31, 1, False, torch.bfloat16),         # no piece keeps 31 pairs apart: the any-size kernel
    (6, 2, 1, 7, 2, 1, False, torch.float16),            # odd head size
    (4, 2, 1, 1024, 512, 8, True, torch.bfloat16),
    (300, 9, 3, 256, 128, 1, False, torch.bfloat16),
    (300, 1, 1, 192, 96, 1, True, torch.float32),
    (130, 16, 2, 128, 64, 1, False, torch.float32),
    (40, 2, 2, 64, 0, 1, False, torch.bfloat16),         # no pairs: the norm alone
    (1500, 2, 1, 32, 16, 1, False, torch.float16),
)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,pairs,axes,interleaved,dtype", CASES)
@pytest.mark.parametrize("eps,weighted", ((1e-6, True), (1e-2, False), (None, False)))
def test_forward_and_gradients(tokens, heads, kv_heads, dim, pairs, axes, interleaved, dtype, eps, weighted):
    q, k, positions, frequencies, gen = make(tokens, heads, kv_heads, dim, pairs, axes, dtype, tokens + dim)
    weights = [None, None]
    if weighted:
        weights = [(1 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).to(dtype).requires_grad_() for _ in range(2)]
    fields = [t.detach().requires_grad_() for t in (q, k)]
    grads = [torch.randn(t.shape, generator=gen, device="cuda").to(dtype) for t in fields]
    out = tg.norm_rotary(*fields, positions, frequencies, query_weight=weights[0], key_weight=weights[1], eps=eps,
                         interleaved=interleaved)
    angle = angles(positions, frequencies)
    half, tiny = HALF[dtype], TINY[dtype]
    with torch.no_grad():                       # the path that builds no graph gives the same bits
        plain = tg.norm_rotary(*fields, positions, frequencies, query_weight=weights[0], key_weight=weights[1],
                               eps=eps, interleaved=interleaved)
    for got, again, x, w in zip(out, plain, fields, weights):
        assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous() and torch.equal(got, again)
        want, magnitude = expected(x.detach(), None if w is None else w.detach(), angle, eps, interleaved)
        assert_within(got, want, half * want.abs() + tiny + 40 * U * magnitude)
    inputs = fields + [w for w in weights if w is not None]
    back = torch.autograd.grad(out, inputs, grads)
    for side, (x, w, dy) in enumerate(zip(fields, weights, grads)):
        x, dy = x.detach().double(), dy.double()
        dn, dn_size = turn(dy, -angle, interleaved), turn_magnitude(dy, pairs, interleaved)
        if eps is None:
            assert_within(back[side], dn, half * dn.abs() + tiny + 40 * U * dn_size)
            continue
        r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        unit = x * r
        scale = 1.0 if w is None else w.detach().double()
        g, g_size = dn * scale, dn_size * (1.0 if w is None else scale.abs())
        want = r * (g - unit * (g * unit).mean(-1, keepdim=True))
        size = r * (g_size + unit.abs() * (g_size * unit.abs()).mean(-1, keepdim=True))
        assert_within(back[side], want, half * want.abs() + tiny + 100 * U * size)
        if w is not None:
            want = (dn * unit).sum((0, 1))
            # added in parts: at most the rows of one warp, 8 warps, and the blocks' partial sums one after the other
            size = (dn_size * unit.abs()).sum((0, 1))
            assert_within(back[2 + side], want, half * want.abs() + tiny + 200 * U * size)


def test_gradients_agree_with_differences():
    q, k, positions, frequencies, gen = make(3, 2, 1, 16, 6, 1, torch.float32, 3, limit=50)
    w = (1 + 0.1 * torch.randn(16, generator=gen, device="cuda")).requires_grad_()
    fields = [t.detach().clone().requires_grad_() for t in (q, k)]
    gradient = [torch.randn(t.shape, generator=gen, device="cuda") for t in fields]

    def loss(*inputs):
        out = tg.norm_rotary(inputs[0], inputs[1], positions, frequencies, query_weight=inputs[2], key_weight=inputs[2])
        return sum((o.double() * g.double()).sum() for o, g in zip(out, gradient))

    inputs = fields + [w]
    back = torch.autograd.grad(loss(*inputs), inputs)
    step = 2.0 ** -7
    for at, (x, g) in enumerate(zip(inputs, back)):
        for index in range(0, x.numel(), 5):
            moved = []
            for sign in (1, -1):
                shifted = [t.detach().clone() for t in inputs]
                shifted[at].view(-1)[index] += sign * step
                moved.append(loss(*shifted).item())
            slope = (moved[0] - moved[1]) / (2 * step)
            # central differences: a third derivative of order 10 times step^2 / 6, and 96 outputs' rounding over 2 steps
            assert abs(slope - g.view(-1)[index].item()) <= 10 * step ** 2 / 6 + 96 * 4 * U / step


def test_far_positions_keep_their_angle():
    """2^40 * 0.9 turns the pair by an angle that float32 could not even hold to a full turn."""
    positions = torch.tensor([2 ** 40 + 12345, -(2 ** 40) - 54321, 2 ** 31 - 1], device="cuda")
    x = torch.randn(3, 2, 8, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    frequencies = torch.tensor([1.0, 0.9, 0.1, 1e-4], device="cuda")
    got, _ = tg.norm_rotary(x, x[:, :1], positions, frequencies, eps=None)
    angle = angles(positions, frequencies)
    want, magnitude = expected(x, None, angle, None, False)
    # the angle itself carries 2^-53 of 2^40: 2^-13 in both computations
    assert_within(got, want, (40 * U + 2.0 ** -12) * magnitude)


def test_strides_alignment_and_a_missing_key():
    gen = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(12, 3, 133, generator=gen, device="cuda").to(torch.bfloat16)
    positions = torch.arange(24, device="cuda", dtype=torch.int32)[::2]
    frequencies = tg.rotary_frequencies(64, device="cuda")
    angle = angles(positions, frequencies)
    views = [base[:, :, :64], base[:, :, 1:65], base[:, :, 3:131:2], base.flip(1)[:, :, 5:69], base[:, ::2, 8:72]]
    for q in views:
        got = tg.norm_rotary(q, None, positions, frequencies)
        want, magnitude = expected(q, None, angle, 1e-6, False)
        assert isinstance(got, torch.Tensor)
        assert_within(got, want, HALF[torch.bfloat16] * want.abs() + 40 * U * magnitude)
    q = views[1].detach().requires_grad_()
    g = torch.randn(12, 64, 3, generator=gen, device="cuda").to(torch.bfloat16).transpose(1, 2)   # strided gradient
    (dx,) = torch.autograd.grad(tg.norm_rotary(q, None, positions, frequencies, eps=None), q, g)
    want = turn(g.double(), -angle, False)
    assert_within(dx, want, HALF[torch.bfloat16] * want.abs() + 40 * U * turn_magnitude(g.double(), 32, False))


def test_values_that_are_not_finite_stay_in_their_head():
    x = torch.randn(4, 3, 64, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    clean = x.clone()
    x[1, 1, 5] = float("nan")
    x[2, 0, 63] = float("inf")                       # not turned: stays an infinity, alone
    positions, frequencies = torch.arange(4, device="cuda"), tg.rotary_frequencies(32, device="cuda")
    got, want = (tg.norm_rotary(t, None, positions, frequencies, eps=None) for t in (x, clean))
    differ = (got != want).nonzero().tolist()
    assert all(p in ([1, 1, 5], [1, 1, 21], [2, 0, 63]) for p in differ)
    assert got[2, 0, 63].item() == float("inf")
    got, want = (tg.norm_rotary(t, None, positions, frequencies) for t in (x, clean))
    assert {tuple(p[:2]) for p in (got != want).nonzero().tolist()} == {(1, 1), (2, 0)}


def test_no_tokens_and_zero_rows():
    frequencies = tg.rotary_frequencies(64, device="cuda")
    empty = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    q, k = tg.norm_rotary(empty, empty[:, :2], torch.empty(0, dtype=torch.int64, device="cuda"), frequencies, query_weight=w)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    dx, dw = torch.autograd.grad(q.sum() + k.sum(), (empty, w))
    assert dx.shape == empty.shape and bool((dw == 0).all())
    zero = torch.zeros(2, 1, 64, device="cuda", requires_grad=True)
    out = tg.norm_rotary(zero, None, torch.tensor([3, 4], device="cuda"), frequencies)
    (dx,) = torch.autograd.grad(out.sum(), zero)
    assert bool((out == 0).all()) and bool(torch.isfinite(dx).all())


def test_weight_gradients_repeat_bit_for_bit():
    q, k, positions, frequencies, gen = make(3001, 4, 2, 64, 32, 1, torch.bfloat16, 9)
    w = torch.ones(64, device="cuda", requires_grad=True)
    fields = [t.detach().requires_grad_() for t in (q, k)]
    runs = []
    for _ in range(3):
        out = tg.norm_rotary(*fields, positions, frequencies, query_weight=w, key_weight=w)
        runs.append(torch.autograd.grad(out[0].float().sum() + out[1].float().square().sum(), w)[0])
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_capture_and_streams():
    q, k, positions, frequencies, gen = make(20, 4, 2, 64, 32, 1, torch.bfloat16, 11)
    q, k = q.contiguous(), k.contiguous()
    eager = tg.norm_rotary(q, k, positions, frequencies)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = tg.norm_rotary(q, k, positions, frequencies)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tg.norm_rotary(q, k, positions, frequencies)
    q.copy_(q.flip(0))
    positions.add_(3)
    graph.replay()
    eager = tg.norm_rotary(q, k, positions, frequencies)
    assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_broadcast_inputs_shared_weights_and_one_output():
    """A query expanded over its heads, one weight for both fields, and a loss that reads one of the outputs."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    base = torch.randn(6, 1, 32, generator=gen, device="cuda", requires_grad=True)
    w = (1 + 0.1 * torch.randn(32, generator=gen, device="cuda")).requires_grad_()
    positions, frequencies = torch.arange(6, device="cuda"), tg.rotary_frequencies(32, device="cuda")
    g = torch.randn(6, 5, 32, generator=gen, device="cuda")
    q, k = tg.norm_rotary(base.expand(6, 5, 32), base, positions, frequencies, query_weight=w, key_weight=w)
    dx, dw = torch.autograd.grad(q, (base, w), g)
    x64, w64 = base.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want, _ = expected(x64.expand(6, 5, 32), w64, angles(positions, frequencies), 1e-6, False)
    rx, rw = torch.autograd.grad(want, (x64, w64), g.double())
    # sums over five heads of values off by 100 u of terms of a few units each
    assert_within(dx, rx, torch.full_like(rx, 5 * 100 * U * 8))
    assert_within(dw, rw, torch.full_like(rw, 30 * 200 * U * 8))


def test_gradients_are_not_differentiable_again():
    x = torch.randn(3, 2, 16, device="cuda", requires_grad=True)
    out = tg.norm_rotary(x, None, torch.arange(3, device="cuda"), tg.rotary_frequencies(16, device="cuda"))
    (dx,) = torch.autograd.grad(out.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), x)


def test_more_heads_than_a_block_and_long_runs():
    """Shares of warps that begin and end inside a token's heads, on both sides."""
    for tokens, heads, kv_heads in ((5, 301, 7), (700, 1, 3), (4099, 3, 1)):
        q, k, positions, frequencies, gen = make(tokens, heads, kv_heads, 64, 32, 1, torch.bfloat16, tokens)
        angle = angles(positions, frequencies)
        fields = [t.detach().requires_grad_() for t in (q, k)]
        out = tg.norm_rotary(*fields, positions, frequencies, eps=1e-5)
        grads = [torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype) for t in out]
        back = torch.autograd.grad(out, fields, grads)
        for x, got, dy, dx in zip(fields, out, grads, back):
            want, magnitude = expected(x.detach(), None, angle, 1e-5, False)
            assert_within(got, want, HALF[torch.bfloat16] * want.abs() + 40 * U * magnitude)
            x, dn, size = x.detach().double(), turn(dy.double(), -angle, False), turn_magnitude(dy.double(), 32, False)
            r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)
            unit = x * r
            want = r * (dn - unit * (dn * unit).mean(-1, keepdim=True))
            size = r * (size + unit.abs() * (size * unit.abs()).mean(-1, keepdim=True))
            assert_within(dx, want, HALF[torch.bfloat16] * want.abs() + 100 * U * size)


def test_far_offsets_of_many_tokens():
    """The last tokens' heads lie behind 2^31 values, in the input and in the output."""
    tokens = 2 ** 31 // (8 * 128) + 50
    q = torch.empty(tokens, 8, 128, device="cuda", dtype=torch.bfloat16)
    q[-70:] = torch.randn(70, 8, 128, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(q.dtype)
    q[:-70] = 1
    positions = torch.arange(tokens, device="cuda", dtype=torch.int32)
    frequencies = tg.rotary_frequencies(128, device="cuda")
    got = tg.norm_rotary(q, None, positions, frequencies)
    want, magnitude = expected(q[-70:], None, angles(positions[-70:], frequencies), 1e-6, False)
    assert_within(got[-70:], want, HALF[q.dtype] * want.abs() + 40 * U * magnitude)
    want, magnitude = expected(q[:70], None, angles(positions[:70], frequencies), 1e-6, False)
    assert_within(got[:70], want, HALF[q.dtype] * want.abs() + 40 * U * magnitude)


def test_a_captured_training_step():
    """Forward and gradients recorded together (no eager graph of the leaves is alive), replayed on new contents."""
    q, k, positions, frequencies, gen = make(50, 4, 2, 64, 32, 1, torch.bfloat16, 21)
    fields = [t.contiguous().detach().requires_grad_() for t in (q, k)]
    weight = torch.ones(64, device="cuda", requires_grad=True)
    grads = [torch.randn(t.shape, generator=gen, device="cuda").to(t.dtype) for t in fields]

    def step():
        out = tg.norm_rotary(*fields, positions, frequencies, query_weight=weight, key_weight=weight)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, fields + [weight], grads))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for i in range(3):
        with torch.no_grad():
            for t in fields + grads + [weight]:
                t.normal_(generator=gen)
            positions.add_(17)
        graph.replay()
        got = [t.clone() for t in recorded]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
