"""GPU: what a vision-language decoder needs around the causal attention of its prompt - rotary positions with several axes, pages
planned on the device, the cache held in 4 bits, attention over it - against plain implementations in 64 bits.

A value rounded to a type is off by at most half a step, finfo(t).eps / 2 relative to it: HALF[t]."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# smallest step of a type's subnormal numbers, halved
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
TYPES = [torch.bfloat16, torch.float16]
names = dict(ids=lambda x: str(x).replace("torch.", "") if isinstance(x, torch.dtype) else None)


@pytest.fixture(scope="module")
def ops():
    from psa_b200 import ops
    assert torch.cuda.is_available()
    yield ops
    ops.check_status()


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


# ---------------------------------------------------------------- rotary positions with several axes
def angles(positions, sections, theta, per_axis, dim):
    """[B, S, D/2] in 64 bits, pair by pair."""
    out, pair = [], 0
    for axis, n in enumerate(sections):
        for j in range(n):
            f = theta ** -(j / n) if per_axis else theta ** -((pair + j) / (dim // 2))
            out.append(positions[axis].double() * f)
        pair += n
    return torch.stack(out, -1)


def turned(x, angle, layout):
    x, c, s = x.double(), torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    u, v = a * c - b * s, b * c + a * s
    return torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)


def pair_size(x, layout):
    """|x0| + |x1| of every channel's pair."""
    x = x.double().abs()
    half = x.shape[-1] // 2
    if layout == "half":
        s = x[..., :half] + x[..., half:]
        return torch.cat([s, s], -1)
    return (x[..., 0::2] + x[..., 1::2]).repeat_interleave(2, -1)


def near_turned(got, x, angle, layout):
    """Cosine and sine: 2^-24 of a half turn from the angle's rounding (pi 2^-25), 2^-22 from the function; three roundings of 2^-24."""
    want = turned(x, angle, layout)
    bound = HALF[x.dtype] * 1.01 * want.abs() + 2.0 ** -21 * pair_size(x, layout) + TINY[x.dtype]
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool(((got.double() - want).abs() <= bound).all())


ROTARY = [  # B, heads, kv heads, S, D, sections, layout, per_axis
    (1, 28, 4, 1, 128, (16, 24, 24), "half", False),
    (2, 7, 1, 77, 128, (16, 24, 24), "half", False),
    (1, 3, 3, 1000, 128, (22, 21, 21), "pairs", True),
    (3, 2, 5, 33, 64, (8, 12, 12), "pairs", True),
    (2, 4, 2, 129, 64, (32,), "half", False),
    (1, 1, 1, 5, 16, (3, 5), "pairs", False),
    (1, 2, 1, 9, 256, (0, 64, 64), "half", True),
    (1, 2, 2, 17, 48, (4, 0, 20), "half", False),
]


@pytest.mark.parametrize("dtype", [*TYPES, torch.float32], **names)
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "x".join(map(str, c[:5])) + c[6])
def test_rotary_axes_turns_and_turns_back(ops, case, dtype):
    B, H, Hk, S, D, sections, layout, per_axis = case
    g = gen(11)
    q, k = randn(g, B, H, S, D, dtype=dtype).requires_grad_(), randn(g, B, Hk, S, D, dtype=dtype).requires_grad_()
    pos = torch.randint(0, 40000, (len(sections), B, S), generator=g, device=DEV)
    ang = angles(pos, sections, 1e4, per_axis, D)
    q2, k2 = ops.rotate_axes(q, k, pos, sections, layout=layout, per_axis=per_axis)
    near_turned(q2.detach(), q.detach(), ang, layout), near_turned(k2.detach(), k.detach(), ang, layout)
    dq2, dk2 = randn(g, B, H, S, D, dtype=dtype), randn(g, B, Hk, S, D, dtype=dtype)
    dq, dk = torch.autograd.grad((q2, k2), (q, k), (dq2, dk2))
    near_turned(dq, dq2, -ang, layout), near_turned(dk, dk2, -ang, layout)
    one = ops.rotate_axes(q.detach(), None, pos.to(torch.int32), sections, layout=layout, per_axis=per_axis)
    assert torch.equal(one, q2.detach())


@pytest.mark.parametrize("far", [0, 131071, 2 ** 31 - 1, -5, 10 ** 12])
def test_rotary_axes_far_positions(ops, far):
    """The product of position and turns is exact modulo one turn; positions beyond 32 bits are off by |pos| 2^-65 turns."""
    x = randn(gen(1), 1, 2, 3, 128)
    pos = torch.tensor([[far, far - 1, far - 77]], device=DEV)
    # the reference in exact arithmetic: whole turns taken off an integer product
    from fractions import Fraction
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    ang = torch.tensor([[float((Fraction(p) * Fraction(1e6 ** -(i / 64)) / two_pi) % 1 * two_pi) for i in range(64)] for p in pos[0].tolist()],
                       dtype=torch.float64, device=DEV)
    near_turned(ops.rotate_axes(x, None, pos, (64,), theta=1e6), x, ang[None], "half")


def test_rotary_axes_views_positions_and_frequencies(ops):
    """Token-major views keep their order; rows that cannot be read in words, expanded rows and expanded gradients are laid out first;
    positions with strides, of one batch element for all, of 32 bits; a table of frequencies instead of theta."""
    g = gen(2)
    B, S, H, D = 2, 50, 6, 64
    base = randn(g, B, S, H, D, dtype=torch.bfloat16)
    pos = torch.randint(0, 9999, (S, B, 3), generator=g, device=DEV).permute(2, 1, 0)
    ang = angles(pos, (8, 12, 12), 1e4, False, D)
    q = base.transpose(1, 2)
    out = ops.rotate_axes(q, None, pos, (8, 12, 12))
    assert out.stride() == q.stride()
    near_turned(out, q, ang, "half")
    fused = randn(g, B, S, 3 * H * D, dtype=torch.bfloat16)
    odd = randn(g, B, H, S, D + 1, dtype=torch.bfloat16)[..., 1:]
    for x in (fused[..., H * D:2 * H * D].unflatten(-1, (H, D)).transpose(1, 2), odd, base.flip(1).transpose(1, 2),
              base[:, :, :1].expand(-1, -1, H, -1).transpose(1, 2), base.permute(0, 3, 1, 2).contiguous().permute(0, 3, 2, 1)):
        near_turned(ops.rotate_axes(x, None, pos, (8, 12, 12)), x, ang, "half")
    same = ops.rotate_axes(q, None, pos[:, :1].to(torch.int32), (8, 12, 12))
    near_turned(same, q, ang[:1], "half")
    assert torch.equal(same, ops.rotate_axes(q, None, pos[:, 0], (8, 12, 12)))
    freq = [0.5 + 0.01 * i for i in range(32)]
    near_turned(ops.rotate_axes(q, None, pos, (32, 0, 0), inv_freq=freq), q, pos[0].double()[..., None] * torch.tensor(freq, dtype=torch.float64, device=DEV), "half")
    leaf = q.detach().clone().requires_grad_()
    ops.rotate_axes(leaf, None, pos, (8, 12, 12)).float().sum().backward()
    near_turned(leaf.grad, torch.ones_like(q), -ang, "half")


def test_rotary_axes_gradients_against_differences(ops):
    """float32: the function is linear, so a central difference is its derivative up to roundings; gradient of the gradient too."""
    g = gen(3)
    q, k = randn(g, 1, 2, 3, 16).requires_grad_(), randn(g, 1, 1, 3, 16).requires_grad_()
    pos = torch.tensor([[0, 3, 50], [7, 7, 9]], device=DEV)
    wq, wk = randn(g, 1, 2, 3, 16), randn(g, 1, 1, 3, 16)

    def f(a, b):
        x, y = ops.rotate_axes(a, b, pos, (3, 5), layout="pairs")
        return (x * wq).double().sum() + (y * wk).double().sum()
    dq, dk = torch.autograd.grad(f(q, k), (q, k))
    for x, d in ((q, dq), (k, dk)):
        for i in range(0, x.numel(), 7):
            step = torch.zeros_like(x).view(-1)
            step[i] = 1.0
            step = step.view_as(x)
            hi = f(q + step, k) if x is q else f(q, k + step)
            lo = f(q - step, k) if x is q else f(q, k - step)
            # values up to about 6, each rounded three times at 2^-24, 16 of them change
            assert abs(float((hi - lo).detach()) / 2 - float(d.view(-1)[i])) < 16 * 6 * 3 * 2.0 ** -24
    # only one of the two wanted; a second derivative
    x, y = ops.rotate_axes(q, k.detach(), pos, (3, 5), layout="pairs")
    assert y.requires_grad is False or torch.autograd.grad(y.sum(), q, allow_unused=True, retain_graph=True)[0] is None
    (d,) = torch.autograd.grad((x * x).sum(), q, create_graph=True)
    (dd,) = torch.autograd.grad(d.sum(), q)
    assert float((dd - 2).abs().max()) < 1e-5        # |R x|^2 = |x|^2


def test_rotary_axes_zero_position_and_empty(ops):
    x = randn(gen(4), 1, 3, 4, 64, dtype=torch.float16)
    x[0, 0, 0, 0], x[0, 1, 1, 5] = 65504.0, 6e-8
    assert torch.equal(ops.rotate_axes(x, None, torch.zeros(1, 4, dtype=torch.int64, device=DEV), (32,)), x)
    e = ops.rotate_axes(x[:, :, :0], x[:, :1, :0], torch.zeros(1, 0, dtype=torch.int64, device=DEV), (32,))
    assert e[0].shape == (1, 3, 0, 64) and e[1].shape == (1, 1, 0, 64)


# ---------------------------------------------------------------- pages
def plan(table, lengths, counts, pool, free, page, tokens):
    """One request after another, on the host."""
    table, lengths, pool = table.tolist(), lengths.tolist(), pool.tolist()
    top, total, taken, slots = free, 0, 0, []
    for b, c in enumerate(counts):
        ok = 0 <= c <= tokens and 0 <= lengths[b] and lengths[b] + c <= len(table[b]) * page
        need = -(-(lengths[b] + c) // page) - -(-lengths[b] // page) if ok else 0
        total += need
        if not ok or (need and total > free):
            c = need = 0
        first = total - need
        held = -(-lengths[b] // page)
        for j in range(need):
            table[b][held + j] = pool[top - 1 - first - j]
        taken = max(taken, first + need) if need else taken
        at = range(lengths[b], lengths[b] + c)
        slots.append([table[b][p // page] * page + p % page for p in at] + [-1] * (tokens - c))
        lengths[b] += c
    return table, lengths, [top - taken], slots


@pytest.mark.parametrize("requests,width,page,tokens,pool", [(1, 1, 16, 1, 3), (5, 9, 16, 40, 60), (70, 33, 64, 300, 900), (1500, 6, 32, 50, 4000),
                                                             (2048, 3, 16, 1, 5000), (3, 4000, 16, 20000, 5000)])
def test_pages_planned_step_by_step(ops, requests, width, page, tokens, pool):
    g = torch.Generator().manual_seed(requests)
    order = torch.randperm(pool, generator=g).to(torch.int32)
    table = torch.full((requests, width), -1, dtype=torch.int32)
    state = [table.to(DEV), torch.zeros(requests, dtype=torch.int32, device=DEV), torch.tensor([pool], dtype=torch.int32, device=DEV)]
    pool_dev = order.to(DEV)
    lengths, free = torch.zeros(requests, dtype=torch.int32), pool
    for step in range(4):
        room = width * page - lengths
        counts = (torch.rand(requests, generator=g) * (torch.minimum(room, torch.tensor(tokens)) + 1)).int()
        counts[torch.rand(requests, generator=g) < 0.2] = 0
        if step == 2:
            counts = torch.minimum(room, torch.ones_like(room)).int()
        want = plan(table, lengths, counts.tolist(), order, free, page, tokens)
        before = [t.clone() for t in state]
        got = ops.plan_pages(*state[:2], counts.to(DEV), pool_dev, state[2], page, tokens)
        assert all(torch.equal(a, b) for a, b in zip(before, state))
        for a, b in zip(got, want):
            assert a.tolist() == b
        inplace = ops.plan_pages(*state[:2], counts.to(DEV).long(), pool_dev, state[2], page, tokens, out=(state[0], state[1], state[2]))
        assert all(torch.equal(a, b) for a, b in zip(inplace, got)) and inplace[0].data_ptr() == state[0].data_ptr()
        refused = int(got[1].sum()) != int(lengths.sum() + counts.sum())
        if refused:
            with pytest.raises(RuntimeError, match="out of range|empty"):
                ops.check_status()
        ops.check_status()
        table, lengths, free = torch.tensor(want[0], dtype=torch.int32), torch.tensor(want[1], dtype=torch.int32), want[2][0]


def test_pages_refused_requests_get_nothing(ops):
    """Counts and lengths out of range, a row that is full, a pool that runs out in the middle: those requests stay as they are."""
    table = torch.full((6, 2), -1, dtype=torch.int32, device=DEV)
    lengths = torch.tensor([0, 31, 0, -3, 99, 1], dtype=torch.int32, device=DEV)
    table[1], table[5, 0] = torch.tensor([7, 8], dtype=torch.int32), 6
    counts = torch.tensor([17, 2, -1, 1, 1, 15], device=DEV)
    pool, free = torch.arange(3, dtype=torch.int32, device=DEV), torch.tensor([9], dtype=torch.int32, device=DEV)   # says more than there are
    t, l, f, s = ops.plan_pages(table, lengths, counts, pool, free, 16, 17)
    assert l.tolist() == [17, 31, 0, -3, 99, 16] and f.tolist() == [1]
    assert t.tolist() == [[2, 1], [7, 8], [-1, -1], [-1, -1], [-1, -1], [6, -1]]
    assert s[0].tolist() == [2 * 16 + i for i in range(16)] + [16] and s[5].tolist() == [6 * 16 + 1 + i for i in range(15)] + [-1] * 2
    assert bool((s[1:5] == -1).all())
    with pytest.raises(RuntimeError):
        ops.check_status()
    # the pool holds 3: the second request's total does not fit, a third that needs none is served, a later one is not
    t, l, f, s = ops.plan_pages(torch.full((4, 4), -1, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV),
                                torch.tensor([32, 33, 0, 1], device=DEV), pool, torch.tensor([3], dtype=torch.int32, device=DEV), 16, 40)
    assert l.tolist() == [32, 0, 0, 0] and f.tolist() == [1]
    with pytest.raises(RuntimeError):
        ops.check_status()


@pytest.mark.parametrize("requests", [1, 40, 1300])
def test_pages_released_in_the_order_that_undoes_them(ops, requests):
    from psa_b200.cache import PageTable
    pt = PageTable(requests, 100, requests * 7 + 3, 16, DEV)
    pool = pt.pool.clone()
    counts = torch.randint(0, 101, (requests,), generator=gen(5), device=DEV)
    pt.reserve(counts, 100)
    assert pt.free.item() == pt.pages - int(((counts + 15) // 16).sum())
    pt.release(torch.ones(requests, dtype=torch.bool, device=DEV))
    assert pt.free.item() == pt.pages and torch.equal(pool, pt.pool) and not bool(pt.lengths.any())
    # some of them: no page is lost or held twice
    pt.reserve(counts, 100)
    some = torch.rand(requests, generator=gen(6), device=DEV) < 0.5
    pt.release(some)
    pt.release(some)                                          # nothing left to give back
    pt.reserve(torch.full((requests,), 3, device=DEV) * some, 3)
    held = [p for row, n in zip(pt.table.tolist(), pt.lengths.tolist()) for p in row[:-(-n // 16)]]
    assert sorted(held + pt.pool[:pt.free.item()].tolist()) == list(range(pt.pages))
    ops.check_status()


# ---------------------------------------------------------------- the cache held in 4 bits
def scales(x, group):
    """step and lowest of every group, as numbers of x's type in 64 bits, and the codes."""
    y = x.double().unflatten(-1, (-1, group))
    low = y.amin(-1, keepdim=True)
    wide = ((y.amax(-1, keepdim=True) - low) / 15)
    step = wide.to(x.dtype)
    step = torch.where(step.double() > wide, (step.view(torch.int16) - 1).view(x.dtype), step).double()
    code = torch.where(step > 0, torch.round((y - low) / torch.where(step > 0, step, 1.0)), 0.0).clamp(0, 15)
    return step, low, code


def stands_for(x, group):
    step, low, code = scales(x, group)
    return (low + code * step).flatten(-2)


def some_slots(g, B, n, pages, page):
    return torch.randperm(pages * page, generator=g, device=DEV)[:B * n].view(B, n).to(torch.int32)


SIZES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("B,H,n,page", [(1, 1, 1, 16), (3, 5, 1, 64), (2, 2, 333, 32), (1, 4, 1029, 128)])
def test_cache_holds_the_nearest_of_16_values(ops, dtype, D, group, B, H, n, page):
    g = gen(D + group + n)
    k = randn(g, B, n, H, D, dtype=dtype).mul_(torch.exp(randn(g, D)).to(dtype)).transpose(1, 2)
    v = randn(g, B, H, n, D, dtype=dtype)
    pages = B * n // page + 2
    data = ops.kv4_empty(pages, H, page, D, group, DEV).random_(0, 256, generator=g)
    before = data.clone()
    slots = some_slots(g, B, n, pages, page)
    skipped = torch.rand(B, n, generator=g, device=DEV) < 0.1
    slots = torch.where(skipped, -1, slots)
    ops.kv4_append(data, k, v, slots, group)
    got = ops.kv4_read(data, slots, D, group, dtype)
    for x, y in zip((k, v), got):
        want = stands_for(x, group)
        keep = ~skipped[:, None].expand(-1, H, -1)
        # the value is the sum of two numbers of the type, rounded to 32 bits and to the type
        assert bool(((y.double() - want).abs()[keep] <= (HALF[dtype] * 1.001 * want.abs() + TINY[dtype])[keep]).all())
        assert bool((y[~keep] == 0).all())
        step, _, _ = scales(x, group)
        worst = (want - x.double()).abs().unflatten(-1, (-1, group)) / step
        assert bool((worst[keep] <= 0.5 + 1e-9).all())
    ops.check_status()
    # every other byte of the cache is as it was: the same rows into a copy with other contents differ in nothing else
    other = ~before
    ops.kv4_append(other, k, v, slots, group)
    written = int((data != ~other).sum())                              # bytes that are no longer each other's inverse
    assert (~skipped).sum().item() * H * (D + 8 * D // group) == written


def test_cache_of_odd_groups(ops):
    """Constant groups, one outlier, smallest and largest numbers, infinities and NaN (the group reads as NaN, its neighbours do not)."""
    for dtype in TYPES:
        big = torch.finfo(dtype).max
        x = randn(gen(7), 1, 1, 9, 64, dtype=dtype)
        x[0, 0, 0] = 3.0
        x[0, 0, 1, 5] = 1000.0
        x[0, 0, 2] *= torch.finfo(dtype).tiny
        x[0, 0, 3, 0], x[0, 0, 3, 1] = (big, -big) if dtype == torch.float16 else (big / 4, -big / 4)
        x[0, 0, 4, 33] = math.inf
        x[0, 0, 5, 3] = math.nan
        x[0, 0, 6, 40] = -math.inf
        x[0, 0, 7] = 0.0
        x[0, 0, 8] = -0.0
        data = ops.kv4_empty(1, 1, 16, 64, 32, DEV)
        slots = torch.arange(9, device=DEV)[None]
        ops.kv4_append(data, x, x.flip(-1), slots, 32)
        k, v = ops.kv4_read(data, slots, 64, 32, dtype)
        bad = torch.zeros(9, 2, dtype=torch.bool, device=DEV)
        bad[4, 1] = bad[5, 0] = bad[6, 1] = True
        assert torch.equal(k[0, 0].unflatten(-1, (2, 32)).isnan().all(-1), bad) and torch.equal(k.isnan().any(-1).sum(), bad.sum())
        assert torch.equal(v[0, 0].unflatten(-1, (2, 32)).isnan().all(-1), bad.flip(-1))
        good = ~bad.repeat_interleave(32, -1)
        want = stands_for(x[0, 0], 32)
        assert bool((k[0, 0].isfinite() == good).all())
        assert bool(((k[0, 0].double() - want).abs() <= HALF[dtype] * 1.001 * want.abs() + TINY[dtype])[good].all())
        assert bool((k[0, 0, 0] == 3).all()) and bool((k[0, 0, 7:] == 0).all())


def test_cache_slots_out_of_range_are_skipped(ops):
    data = torch.zeros_like(ops.kv4_empty(2, 1, 16, 64, 32, DEV))
    k = randn(gen(8), 1, 1, 4, 64, dtype=torch.float16)
    slots = torch.tensor([[32, -2, 2 ** 30, 31]], device=DEV)
    ops.kv4_append(data, k, k, slots, 32)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert not bool(data[0].any()) and bool(data[1].any())
    got = ops.kv4_read(data, slots, 64, 32, torch.float16)[0]
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert not bool(got[0, 0, :3].any()) and bool(got[0, 0, 3].any())
    ops.kv4_append(data, k[:, :, :0], k[:, :, :0], slots[:, :0], 32)
    assert ops.kv4_read(data, slots[:, :0], 64, 32, torch.float16)[1].shape == (1, 1, 0, 64)
    ops.check_status()


# ---------------------------------------------------------------- attention over it
class Filled:
    """A cache with requests of given lengths on pages in no order; rows behind a length, and pages nobody holds, hold any bytes."""

    def __init__(self, ops, g, lengths, Hk, D, group, dtype, page, spare=3, k_scale=1.0, v_scale=1.0, width=None):
        self.lengths, self.D, self.group, self.dtype, self.page, B = lengths, D, group, dtype, page, len(lengths)
        longest = max(max(lengths), 1)
        self.k = (randn(g, B, Hk, longest, D) * torch.exp(0.4 * randn(g, D)) * k_scale + 0.4 * randn(g, D)).to(dtype)
        self.v = (randn(g, B, Hk, longest, D) * torch.exp(0.3 * randn(g, D)) * v_scale).to(dtype)
        held = [-(-n // page) for n in lengths]
        pages = sum(held) + spare
        order = torch.randperm(pages, generator=g, device=DEV).tolist()
        width = max(max(held), 1) if width is None else width
        rows, slots = [], torch.full((B, longest), -1, dtype=torch.int32)
        for b, n in enumerate(held):
            mine = [order.pop() for _ in range(n)]
            rows.append(mine + [-1] * (width - n))
            for t in range(lengths[b]):
                slots[b, t] = mine[t // page] * page + t % page
        self.table = torch.tensor(rows, dtype=torch.int32, device=DEV)
        self.data = ops.kv4_empty(pages, Hk, page, D, group, DEV).random_(0, 256, generator=g)
        self.slots = slots.to(DEV)
        ops.kv4_append(self.data, self.k, self.v, self.slots, group)
        self.len = torch.tensor(lengths, dtype=torch.int32, device=DEV)


def attention(q, c, counts=None, scale=None):
    """-> outputs, logarithms of sums and the bound of the outputs' error, in 64 bits."""
    B, H, n, D = q.shape
    Hk = c.k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, lse, tol, lse_tol = (torch.zeros(B, H, n, m, dtype=torch.float64, device=DEV) for m in (D, 1, D, 1))
    k, v = stands_for(c.k, c.group), stands_for(c.v, c.group)
    k_step = scales(c.k, c.group)[0].amax()
    v_step = scales(c.v, c.group)[0].expand(*c.v.shape[:-1], -1, c.group).flatten(-2)
    for b in range(B):
        count = n if counts is None else counts[b]
        at = c.lengths[b] - count + torch.arange(n, device=DEV)
        at = torch.where(torch.arange(n, device=DEV) < count, at, -1)
        L = c.lengths[b]
        kk, vv, step = (x[b, :, :L].repeat_interleave(H // Hk, 0) for x in (k, v, v_step))
        s = q[b].double() @ kk.transpose(-1, -2) * scale
        s = s.masked_fill(torch.arange(L, device=DEV) > at[:, None], -math.inf)
        m = s.amax(-1, keepdim=True) if L else torch.full((H, n, 1), -math.inf, dtype=torch.float64, device=DEV)
        p = torch.exp(s - m.clamp(min=-1e300))
        total = p.sum(-1, keepdim=True)
        p = p / total.clamp(min=1e-300)
        out[b], lse[b] = p @ vv, m + torch.log(total)
        # a score is a sum over the channels of q times a code times a step, in 32 bits - 2^-21 of the terms' sum, where a code and what
        # is taken off it again come to 143 at most - and of the sum of q, in two terms of 8 bits (2^-17), times a lowest value
        size = q[b].double().abs().sum(-1, keepdim=True)
        off = abs(scale) * size * (2.0 ** -21 * 143 * k_step + 2.0 ** -17 * (kk.abs().amax() if L else 0))
        off = off + 2.0 ** -22 * (1 + s.masked_fill(s == -math.inf, 0).abs().amax(-1, keepdim=True) if L else 1)
        # a weight times a step is rounded to f16, half a step of which is 2^-11, and meets a code less 8; products and sums in 32 bits
        tol[b] = HALF[q.dtype] * 1.01 * out[b].abs() + (2 * off + 2.0 ** -16) * (p @ vv.abs()) + 2.0 ** -11 * (p @ (8 * step)) + TINY[q.dtype]
        lse_tol[b] = off + 2.0 ** -17 + 2.0 ** -23 * lse[b].abs().nan_to_num(0, 0, 0)
    return out, lse[..., 0], tol, lse_tol[..., 0]


def check_attention(ops, q, c, counts=None, scale=None):
    count = None if counts is None else torch.tensor(counts, device=DEV)
    got, lse = ops.kv4_attention(q, c.data, c.table, c.len, c.group, count, scale, return_lse=True)
    want, want_lse, tol, lse_tol = attention(q, c, counts, scale)
    assert got.shape == q.shape and got.dtype == q.dtype and bool(got.isfinite().all())
    far = (got.double() - want).abs() / tol
    assert float(far.max()) <= 1, f"{float(far.max())} of the bound at {far.argmax().item()}"
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty) and bool((got[empty] == 0).all())
    assert bool(((lse.double() - want_lse).abs()[~empty] <= lse_tol[~empty]).all())
    ops.check_status()
    return got


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("H,Hk,n,lengths", [(1, 1, 1, [1]), (7, 1, 1, [1, 15, 16, 17, 0, 63, 64, 65]), (28, 4, 1, [500, 3, 129]), (6, 2, 3, [3, 4, 700, 64]),
                                            (16, 16, 1, [33, 1000]), (9, 1, 5, [5, 77, 2000]), (8, 4, 40, [40, 41, 333])])
def test_attention_over_the_cache(ops, dtype, D, group, H, Hk, n, lengths):
    g = gen(D + group + H + n)
    c = Filled(ops, g, lengths, Hk, D, group, dtype, 64 if H % 2 else 16)
    check_attention(ops, randn(g, len(lengths), n, H, D, dtype=dtype).transpose(1, 2), c)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 272])
def test_attention_pages_of_other_sizes(ops, page):
    """Pages smaller, larger and not a multiple of a tile; lengths at their borders."""
    g = gen(page)
    lengths = [page - 1, page, page + 1, 3 * page, 3 * page + 17, 1]
    c = Filled(ops, g, lengths, 2, 128, 32, torch.bfloat16, page, width=7)
    check_attention(ops, randn(g, 6, 14, 2, 128, dtype=torch.bfloat16), c)


@pytest.mark.parametrize("dtype", TYPES, **names)
def test_attention_counts_of_a_padded_batch(ops, dtype):
    """Requests with fewer new tokens than rows, with none, and with more than they have tokens (rows before the first key)."""
    g = gen(21)
    lengths = [200, 64, 5, 0, 1, 90]
    c = Filled(ops, g, lengths, 2, 64, 32, dtype, 32)
    got = check_attention(ops, randn(g, 6, 6, 8, 64, dtype=dtype), c, counts=[3, 8, 8, 8, 1, 0])
    assert not bool(got[0, :, 3:].any()) and not bool(got[3].any()) and not bool(got[5].any()) and not bool(got[2, :, :3].any())
    assert bool(got[2, :, 3].any())


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(6.0, 2.0, 1.0), (1.0, 1.0, 200.0), (0.02, 0.02, 1e-3), (20.0, 3.0, 0.1)])
def test_attention_of_sharp_flat_large_and_small_values(ops, dtype, q_scale, k_scale, v_scale):
    g = gen(23)
    c = Filled(ops, g, [3000, 64, 1], 2, 128, 64, dtype, 64, k_scale=k_scale, v_scale=v_scale)
    check_attention(ops, randn(g, 3, 8, 1, 128).mul_(q_scale).to(dtype), c)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_attention_scales(ops, scale):
    g = gen(24)
    c = Filled(ops, g, [300, 20], 1, 64, 64, torch.float16, 16)
    check_attention(ops, randn(g, 2, 3, 2, 64, dtype=torch.float16), c, scale=scale)


def test_attention_maximum_that_rises_late_and_falls(ops):
    """Keys that line up with the query more and more, and less and less: the running maximum moves all the way, or never."""
    g = gen(25)
    c = Filled(ops, g, [2000, 2000], 1, 128, 32, torch.bfloat16, 64)
    u = randn(g, 128, dtype=torch.bfloat16)
    ramp = torch.linspace(-3, 3, 2000, device=DEV)[:, None].to(torch.bfloat16)
    c.k[0, 0], c.k[1, 0] = u * ramp, u * -ramp
    ops.kv4_append(c.data, c.k, c.v, c.slots, 32)
    check_attention(ops, (u * 1.5).expand(2, 4, 1, 128).clone(), c)


def test_attention_is_blind_to_what_it_does_not_see(ops):
    """NaN and infinities behind a length, in pages that nobody holds and in later tokens of the same call change nothing; in a key or a
    value that a row sees they do."""
    g = gen(26)
    for H, n in ((7, 4), (1, 1), (3, 11)):
        c = Filled(ops, g, [150, 64, 20], 1, 128, 32, torch.bfloat16, 64)
        q = randn(g, 3, H, n, 128, dtype=torch.bfloat16)
        clean = ops.kv4_attention(q, c.data, c.table, c.len, 32)
        dirty = torch.full_like(c.data, 0xff)                       # every parameter a NaN
        dirty_slots = c.slots
        ops.kv4_append(dirty, c.k, c.v, dirty_slots, 32)
        assert torch.equal(ops.kv4_attention(q, dirty, c.table, c.len, 32), clean)
        # the last token's key and value
        for what in ("k", "v"):
            x = getattr(c, what).clone()
            x[0, 0, 149, 40] = math.nan
            x[1, 0, 63, 3] = math.inf
            ops.kv4_append(c.data, x if what == "k" else c.k, x if what == "v" else c.v, c.slots, 32)
            got = ops.kv4_attention(q, c.data, c.table, c.len, 32)
            assert torch.equal(got[:, :, :n - 1], clean[:, :, :n - 1]) and torch.equal(got[2], clean[2])
            last = got[:2, :, n - 1].isnan()
            if what == "k":
                assert bool(last.all())
            else:
                want = torch.zeros_like(last)
                want[0, :, 32:64] = True
                want[1, :, :32] = True
                assert torch.equal(last, want)
            ops.kv4_append(c.data, c.k, c.v, c.slots, 32)
    ops.check_status()


def test_attention_skips_pages_and_lengths_out_of_range(ops):
    """A page number that the cache does not have hides its tokens; a length beyond the table's row is cut to it; both are reported."""
    g = gen(27)
    c = Filled(ops, g, [64, 64], 1, 64, 32, torch.float16, 16)
    q = randn(g, 2, 2, 1, 64, dtype=torch.float16)
    bad = c.table.clone()
    bad[0, 1], bad[1, 3] = 10 ** 6, -7
    got = ops.kv4_attention(q, c.data, bad, c.len, 32)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    v = stands_for(c.v, 32)
    k = stands_for(c.k, 32)
    for b, gone in ((0, slice(16, 32)), (1, slice(48, 64))):
        s = q[b].double() @ k[b].transpose(-1, -2) / 8
        s[..., gone] = -math.inf
        want = torch.softmax(s, -1) @ v[b]
        assert float((got[b].double() - want).abs().max()) < 2e-3
    assert torch.equal(ops.kv4_attention(q, c.data, c.table, c.len + 1000, 32), ops.kv4_attention(q, c.data, c.table, c.len, 32))
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert not bool(ops.kv4_attention(q, c.data, c.table, c.len - 1000, 32).any())
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()


def test_attention_views_and_repeats(ops):
    """Any order of q's dimensions, rows that cannot be read in words, and bit-equal repeats."""
    g = gen(28)
    c = Filled(ops, g, [777, 100, 3], 2, 64, 64, torch.bfloat16, 32)
    q = randn(g, 3, 2, 10, 64, dtype=torch.bfloat16).transpose(1, 2)
    first = check_attention(ops, q, c)
    assert first.stride() == q.stride()
    odd = torch.empty(3, 10, 2, 65, dtype=q.dtype, device=DEV)[..., 1:]
    odd.copy_(q)
    for x in (q.contiguous(), odd, q, q):
        assert torch.equal(ops.kv4_attention(x, c.data, c.table, c.len, 64), first)
    assert ops.kv4_attention(q[:, :, :0], c.data, c.table, c.len, 64).shape == (3, 10, 0, 64)


def test_attention_of_a_long_context_and_many_requests(ops):
    """Split over many blocks: one long request, and more requests than blocks."""
    g = gen(29)
    c = Filled(ops, g, [70001], 1, 128, 32, torch.bfloat16, 64)
    check_attention(ops, randn(g, 1, 7, 1, 128, dtype=torch.bfloat16), c)
    c = Filled(ops, g, [(i * 37) % 300 for i in range(700)], 2, 64, 32, torch.float16, 16)
    check_attention(ops, randn(g, 700, 4, 1, 64, dtype=torch.float16), c)


def test_cache_offsets_beyond_32_bits(ops):
    """A cache of more than 2^32 bytes: its last page, written, read and attended to."""
    pages = (1 << 32) // (64 * 160 * 4) + 9
    data = ops.kv4_empty(pages, 4, 64, 128, 32, DEV)
    g = gen(30)
    k, v = (randn(g, 1, 4, 64, 128, dtype=torch.bfloat16) for _ in range(2))
    slots = ((pages - 1) * 64 + torch.arange(64, device=DEV))[None]
    assert data.numel() > 1 << 32
    ops.kv4_append(data, k, v, slots, 32)
    assert float((ops.kv4_read(data, slots, 128, 32, torch.bfloat16)[1].double() - stands_for(v, 32)).abs().max()) < 0.02
    q = randn(g, 1, 8, 1, 128, dtype=torch.bfloat16)
    got = ops.kv4_attention(q, data, torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV), torch.tensor([64], dtype=torch.int32, device=DEV), 32)
    kk, vv = (stands_for(x, 32)[0].repeat_interleave(2, 0) for x in (k, v))
    want = torch.softmax(q[0].double() @ kk.transpose(-1, -2) * 128 ** -0.5, -1) @ vv
    assert float((got[0].double() - want).abs().max()) < 0.02
    ops.check_status()


# ---------------------------------------------------------------- more than 16 rows a key head
MANY = [(10, 2, 5, [5, 70, 3000]), (4, 1, 8, [9, 64, 65, 8]), (6, 1, 8, [1000, 8]), (28, 4, 6, [4000, 77]), (8, 8, 20, [20, 500, 33]), (7, 1, 64, [64, 900])]


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
@pytest.mark.parametrize("H,Hk,n,lengths", MANY)
def test_attention_of_many_rows(ops, dtype, D, group, H, Hk, n, lengths):
    g = gen(2 * D + group + H + n)
    c = Filled(ops, g, lengths, Hk, D, group, dtype, 64 if n % 2 else 128)
    check_attention(ops, randn(g, len(lengths), n, H, D, dtype=dtype).transpose(1, 2), c)


@pytest.mark.parametrize("page", [16, 48, 272])
@pytest.mark.parametrize("n", [4, 8])
def test_attention_of_many_rows_pages_of_other_sizes(ops, page, n):
    """Pages that do not hold whole tiles, a copy a slice; more than 8 tiles of them, and lengths at their borders."""
    g = gen(page + n)
    lengths = [max(page - 1, n), page + n, 3 * page + 17, n, 1500, 700]
    c = Filled(ops, g, lengths, 2, 128, 32, torch.float16, page)
    check_attention(ops, randn(g, 6, 14, n, 128, dtype=torch.float16), c)


@pytest.mark.parametrize("n", [3, 6])
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(6.0, 2.0, 1.0), (1.0, 1.0, 200.0), (0.02, 0.02, 1e-3), (20.0, 3.0, 0.1)])
def test_attention_of_many_rows_sharp_flat_large_and_small(ops, n, q_scale, k_scale, v_scale):
    g = gen(33)
    c = Filled(ops, g, [3000, 64, 6], 2, 128, 64, torch.bfloat16, 64, k_scale=k_scale, v_scale=v_scale)
    check_attention(ops, randn(g, 3, 16, n, 128).mul_(q_scale).to(torch.bfloat16), c)


def test_attention_of_many_rows_maximum_that_rises_late_and_falls(ops):
    """The references of all warps move together: keys that line up with some rows' queries more and more, with others' less and less."""
    g = gen(34)
    c = Filled(ops, g, [2000, 2000], 1, 128, 32, torch.bfloat16, 64)
    u = randn(g, 128, dtype=torch.bfloat16)
    ramp = torch.linspace(-3, 3, 2000, device=DEV)[:, None].to(torch.bfloat16)
    c.k[0, 0], c.k[1, 0] = u * ramp, u * -ramp
    ops.kv4_append(c.data, c.k, c.v, c.slots, 32)
    sign = torch.where(torch.arange(12, device=DEV) % 3 == 0, -1.0, 1.0).to(torch.bfloat16)[None, :, None, None]
    check_attention(ops, (u * 1.5 * sign).expand(2, 12, 3, 128).clone(), c)


@pytest.mark.parametrize("dtype", TYPES, **names)
def test_attention_of_many_rows_counts_and_scales(ops, dtype):
    """Requests with fewer new tokens than rows, none, and more than they have tokens; scales of either sign and none."""
    g = gen(35)
    c = Filled(ops, g, [200, 64, 5, 0, 1, 90], 2, 64, 32, dtype, 32)
    q = randn(g, 6, 6, 11, 64, dtype=dtype)
    for scale in (None, 0.0, -0.3):
        got = check_attention(ops, q, c, counts=[3, 11, 11, 11, 1, 0], scale=scale)
    assert not bool(got[0, :, 3:].any()) and not bool(got[3].any()) and not bool(got[5].any()) and not bool(got[2, :, :6].any())


# ---------------------------------------------------------------- all of it together
class Layer:
    """One attention layer of a decoder: rotary positions with three axes, the new keys and values into the cache, attention over it."""

    def __init__(self, table, Hk, D, dtype, group):
        from psa_b200.cache import KV4Cache
        self.cache = KV4Cache(table, Hk, D, dtype, group)
        self.k, self.v = [], []                                   # what every request holds, as it was appended

    def step(self, ops, q, k, v, positions, slots, counts):
        q, k = ops.rotate_axes(q, k, positions, (8, 12, 12) if q.shape[-1] == 64 else (16, 24, 24), theta=1e6)
        self.cache.append(k, v, slots)
        return q, k, self.cache.attend(q, counts)


def token_major(g, B, n, H, D, dtype):
    return randn(g, B, n, H, D, dtype=dtype).transpose(1, 2)


@pytest.mark.parametrize("dtype,D,group,H,Hk", [(torch.bfloat16, 128, 32, 28, 4), (torch.float16, 64, 64, 6, 6)], **names)
def test_answering_prompts_and_tokens(ops, dtype, D, group, H, Hk):
    """Prompts of different lengths in one padded batch, single tokens, drafted tokens, a request that ends and another in its place:
    every output against plain attention in 64 bits over what the cache stands for."""
    from psa_b200.cache import PageTable
    g = gen(40)
    B = 4
    table = PageTable(B, 400, 40, 32, DEV)
    layers = [Layer(table, Hk, D, dtype, group) for _ in range(2)]
    held = [[(torch.zeros(Hk, 0, D, dtype=dtype, device=DEV),) * 2 for _ in range(B)] for _ in layers]
    for counts in ([150, 3, 77, 0], [1, 1, 1, 0], [1, 1, 1, 31], [5, 0, 2, 5], "end 1", [1, 40, 1, 1], [1, 1, 1, 1]):
        if counts == "end 1":
            table.release(torch.tensor([False, True, False, False], device=DEV))
            for h in held:
                h[1] = (torch.zeros(Hk, 0, D, dtype=dtype, device=DEV),) * 2
            continue
        n = max(counts)
        count = torch.tensor(counts, device=DEV)
        start = table.lengths.clone()
        slots = table.reserve(count, n)
        pos = (start[:, None] + torch.arange(n, device=DEV)).expand(3, B, n)
        for layer, h in zip(layers, held):
            q, k, v = (token_major(g, B, n, heads, D, dtype) for heads in (H, Hk, Hk))
            q, k, out = layer.step(ops, q, k, v, pos, slots, count)
            for b, m in enumerate(counts):
                h[b] = tuple(torch.cat([old, new[b, :, :m]], 1) for old, new in zip(h[b], (k, v)))
            longest = max(x[0].shape[1] for x in h)

            class Held:
                pass
            c = Held()
            c.group, c.lengths = group, [x[0].shape[1] for x in h]
            c.k, c.v = (torch.stack([torch.nn.functional.pad(x[i], (0, 0, 0, longest - x[i].shape[1])) for x in h]) for i in (0, 1))
            assert table.lengths.tolist() == c.lengths
            want, _, tol, _ = attention(q, c, counts)
            assert bool(((out.double() - want).abs() <= tol).all())
    ops.check_status()


def test_answering_step_captured_and_replayed(ops):
    """One step of two layers as a CUDA graph, replayed with other tokens, against the same steps launched one by one; a second graph of the
    same state between them."""
    from psa_b200.cache import PageTable
    g = gen(41)
    B, H, Hk, D, dtype = 3, 8, 2, 64, torch.bfloat16

    def state():
        table = PageTable(B, 300, 60, 16, DEV)
        return table, [Layer(table, Hk, D, dtype, 32) for _ in range(2)]
    eager, replayed = state(), state()
    inputs = [token_major(g, B, 1, heads, D, dtype) for heads in (H, Hk, Hk)]
    drafted = [token_major(g, B, 4, heads, D, dtype) for heads in (4 * H, Hk, Hk)]
    ones, four = torch.ones(B, dtype=torch.int32, device=DEV), torch.tensor([4, 0, 3], dtype=torch.int32, device=DEV)

    def step(s, xs, counts):
        table, layers = s
        n = xs[0].shape[2]
        start = table.lengths.clone()
        slots = table.reserve(counts, n)
        pos = (start[:, None] + torch.arange(n, device=DEV, dtype=torch.int32)).expand(3, B, n)
        return [layer.step(ops, *xs, pos, slots, counts)[2] for layer in layers]
    for s in (eager, replayed):                                    # a start, and every kernel's first launch outside the captures
        step(s, [x.expand(-1, -1, 90, -1).contiguous() if x.shape[2] == 1 else x for x in inputs], torch.tensor([90, 17, 64], device=DEV))
        step(s, drafted, four)
    graphs, outs = [], []
    for xs, counts in ((inputs, ones), (drafted, four)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(replayed, xs, counts))
        graphs.append(graph)
    for which in (0, 0, 1, 0, 1, 1, 0):
        for x in (inputs, drafted)[which]:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV).to(dtype))
        want = step(eager, (inputs, drafted)[which], (ones, four)[which])
        graphs[which].replay()
        assert all(torch.equal(a, b) for a, b in zip(outs[which], want))
    assert torch.equal(eager[0].lengths, replayed[0].lengths) and torch.equal(eager[0].table, replayed[0].table)
    ops.check_status()


def test_rotary_backward_captured(ops):
    """Forward and gradients in a captured graph, replayed with other values.  (No eager graph of the same leaves is alive while it is
    captured: PyTorch's engine would make its stream wait for the capturing one, whatever the operator, and the capture would fail.)"""
    g = gen(42)
    q, k = (token_major(g, 1, 33, h, 64, torch.bfloat16).requires_grad_() for h in (4, 2))
    pos = torch.arange(33, dtype=torch.int32, device=DEV)[None]
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def both():
        outs = ops.rotate_axes(q, k, pos, (32,))
        return [x.detach() for x in outs], torch.autograd.grad(outs, (q, k), (dq, dk))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs, grads = both()
    for _ in range(2):
        dq.copy_(torch.randn_like(dq)), dk.copy_(torch.randn_like(dk))
        with torch.no_grad():
            q.copy_(torch.randn_like(q)), k.copy_(torch.randn_like(k))
        graph.replay()
        want_outs, want = both()
        assert all(torch.equal(a, b) for a, b in zip((*outs, *grads), (*want_outs, *want)))


def test_answering_on_other_streams_and_threads(ops):
    """Calls on a stream of their own, and from several host threads at once, give what they give one after another."""
    import threading
    g = gen(43)
    cases = []
    for i in range(4):
        c = Filled(ops, g, [300 + 100 * i, 40, 1000], 2, 64 if i % 2 else 128, 32, TYPES[i // 2], 64)
        q = randn(g, 3, 2 * (1, 4, 9, 20)[i], 1, c.D, dtype=c.dtype)
        pos = torch.arange(len(c.lengths), device=DEV).view(1, 3, 1).int()
        cases.append((c, q, pos))

    def call(c, q, pos):
        turned = ops.rotate_axes(q, None, pos, (c.D // 2,))
        return ops.kv4_attention(turned, c.data, c.table, c.len, c.group), *ops.kv4_read(c.data, c.slots, c.D, c.group, c.dtype)
    want = [call(*x) for x in cases]
    torch.cuda.synchronize()
    got, failed = [None] * len(cases), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = call(*cases[i])
            stream.synchronize()
        except Exception as e:          # noqa: BLE001  (reported by the main thread)
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    ops.check_status()


@pytest.mark.parametrize("H", [1, 2, 3, 6])
@pytest.mark.parametrize("dtype", TYPES, **names)
def test_cache_of_few_heads(ops, H, dtype):
    """A thread's four rows are of one, two or four tokens, over the ends of batch elements; some slots are none."""
    g = gen(44 + H)
    B, n, D = 3, 7, 64
    k, v = token_major(g, B, n, H, D, dtype), randn(g, B, H, n, D, dtype=dtype)
    data = ops.kv4_empty(3, H, 16, D, 32, DEV)
    slots = some_slots(g, B, n, 3, 16)
    slots[1, 3] = slots[2, 6] = -1
    ops.kv4_append(data, k, v, slots, 32)
    for x, y in zip((k, v), ops.kv4_read(data, slots, D, 32, dtype)):
        want = stands_for(x, 32) * (slots >= 0)[:, None, :, None]
        assert bool(((y.double() - want).abs() <= HALF[dtype] * 1.001 * want.abs() + TINY[dtype]).all())
    ops.check_status()


@pytest.mark.parametrize("dtype", TYPES, **names)
def test_cache_ties_go_to_the_even_code(ops, dtype):
    """Values exactly between two codes, for steps whose inverse is rounded: lowest 0, step s, values (i + 1/2) s."""
    steps = [1.0, 3.0, 5.0, 7.0, 11.0, 13.0, 0.375, 49.0]
    x = torch.zeros(1, 1, len(steps), 64, device=DEV)
    for t, s in enumerate(steps):
        x[0, 0, t, :15] = (torch.arange(15, device=DEV) + 0.5) * s
        x[0, 0, t, 16], x[0, 0, t, 32:48] = 15 * s, torch.arange(16, device=DEV) * s
    x = x.to(dtype)
    exact = (x.double()[..., :15] == ((torch.arange(15, device=DEV) + 0.5) * torch.tensor(steps, device=DEV)[:, None]).double()).all(-1)[0, 0]
    # (2 i + 1) s / 2 up to 29 s / 2: whole numbers of s's last place up to 29 s, which bf16 (8 bits) holds up to s = 7 (and 3 / 8), f16 all
    assert int(exact.sum()) == (5 if dtype == torch.bfloat16 else 8)
    data = ops.kv4_empty(1, 1, 16, 64, 64, DEV)
    slots = torch.arange(len(steps), device=DEV)[None]
    ops.kv4_append(data, x, x, slots, 64)
    k, v = ops.kv4_read(data, slots, 64, 64, dtype)
    want = stands_for(x, 64)
    for y in (k, v):
        assert bool(((y.double() - want).abs() <= HALF[dtype] * 1.001 * want.abs()).all())


@pytest.mark.parametrize("H,n", [(7, 1), (12, 1), (10, 3)])
@pytest.mark.parametrize("v_scale", [1e-20, 1e-12, 1e20, 1e29])
def test_attention_of_very_large_and_small_values(ops, H, n, v_scale):
    """Weights times steps stay within f16 wherever the steps are: the references take them along."""
    g = gen(50)
    c = Filled(ops, g, [900, 64, 5], 1, 64, 32, torch.bfloat16, 32, v_scale=v_scale)
    check_attention(ops, randn(g, 3, H, n, 64, dtype=torch.bfloat16), c)


def test_rotary_axes_gradients_of_any_layout(ops):
    """Operands and gradients that cannot be read word by word, or are broadcast, in both orders; k without a gradient, q without one;
    a second derivative through both operands."""
    g = gen(51)
    pos = torch.randint(0, 999, (2, 2, 9), generator=g, device=DEV)
    ang = angles(pos, (12, 20), 1e4, False, 64)
    odd = randn(g, 2, 3, 9, 65, dtype=torch.bfloat16).requires_grad_()
    k = randn(g, 2, 9, 2, 64, dtype=torch.bfloat16).transpose(1, 2).detach().requires_grad_()
    for q in (odd[..., 1:], odd[..., :64].contiguous()):
        x, y = ops.rotate_axes(q, k, pos, (12, 20))
        near_turned(x.detach(), q.detach(), ang, "half")
        up = randn(g, 2, 1, 9, 1, dtype=torch.bfloat16).expand(-1, 3, -1, 64)
        down = randn(g, 2, 2, 64, 9, dtype=torch.bfloat16).transpose(2, 3)
        dq, dk = torch.autograd.grad((x, y), (q, k), (up, down), retain_graph=True)
        near_turned(dq, up, -ang, "half"), near_turned(dk, down, -ang, "half")
        (only,) = torch.autograd.grad(y, k, down, retain_graph=True)
        assert torch.equal(only, dk)
        x, y = ops.rotate_axes(q.detach(), k, pos, (12, 20))
        assert torch.equal(torch.autograd.grad((x, y), k, (up, down))[0], dk)
        x, y = ops.rotate_axes(q, k.detach(), pos, (12, 20))
        assert torch.equal(torch.autograd.grad((x, y), q, (up, down))[0], dq)
    a, b = randn(g, 2, 3, 9, 64).requires_grad_(), randn(g, 2, 2, 9, 64).requires_grad_()
    x, y = ops.rotate_axes(a, b, pos, (12, 20), layout="pairs")
    da, db = torch.autograd.grad((x.pow(3).sum() + y.pow(2).sum()), (a, b), create_graph=True)
    (daa,) = torch.autograd.grad(da.sum(), a)
    # d/da sum(R^T 3 (R a)^2) = R^T (6 (R a) * R 1)
    ones = torch.ones_like(a)
    r1 = turned(ones, ang, "pairs")
    want = turned(6 * turned(a.detach(), ang, "pairs") * r1, -ang, "pairs")
    assert float((daa.double() - want).abs().max()) < 2.0 ** -18 * float(want.abs().max())      # four rotations, 2^-21 each (near_turned)
    assert float((db.detach() - 2 * b.detach()).abs().max()) < 2.0 ** -17                       # R^T 2 R b; |b| up to about 5
    ops.check_status()


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("H,n", [(3, 1), (12, 1), (7, 3), (10, 3), (12, 4)])
def test_attention_skips_bad_pages_wherever_they_are(ops, page, H, n):
    """Page numbers that the cache does not have, alone and next to each other, first and last of a request: their tokens are hidden, all
    others' outputs are those without them; a request of bad pages alone gives rows of nothing."""
    g = gen(60 + page)
    c = Filled(ops, g, [700, 130, 900, 60], 1, 128, 64, torch.bfloat16, page)
    q = randn(g, 4, H, n, 128, dtype=torch.bfloat16)
    bad = c.table.clone()
    for b, entries in ((0, (0, 2, 3, 4)), (1, (1,)), (2, (1, 3, 6))):
        for e in entries:
            if e * page < c.lengths[b]:
                bad[b, e] = (-1, 10 ** 6, c.data.shape[0])[e % 3]
    bad[3] = -5
    got, lse = ops.kv4_attention(q, c.data, bad, c.len, 64, return_lse=True)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    k, v = (stands_for(x, 64)[:, 0] for x in (c.k, c.v))
    for b in range(4):
        L = c.lengths[b]
        hidden = ((bad[b] < 0) | (bad[b] >= c.data.shape[0])).repeat_interleave(page)[:L]
        s = q[b].double() @ k[b, :L].T * 128 ** -0.5
        s = s.masked_fill(hidden | (torch.arange(L, device=DEV) > L - n + torch.arange(n, device=DEV)[:, None]), -math.inf)
        if bool(hidden.all()):
            assert not bool(got[b].any()) and bool((lse[b] == -math.inf).all())
            continue
        want = torch.softmax(s, -1) @ v[b, :L]
        size = torch.softmax(s, -1) @ v[b, :L].abs()
        # bf16's half step, the weights' 2^-11 on what the codes add (at most 8 / 15 of a group's range, twice the values' size), scores to 2^-9
        assert bool(((got[b].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * size + 2.0 ** -10 * v[b, :L].abs().amax()).all())
    assert not bool(got.isnan().any())
