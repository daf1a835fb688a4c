"""GPU: the ends of the ranges that the operators around the causal attention of a prompt promise - sums of many bits, constant and
far values, large pages, long rows - against plain implementations in 64 bits.  (test_gpu_answering.py has the ordinary sizes.)"""
import math

import pytest
import torch

from test_gpu_answering import (DEV, HALF, SIZES, TINY, TYPES, Filled, angles, attention, check_attention, gen, names, near_turned, ops, randn, scales,  # noqa: F401
                                stands_for)

pytestmark = pytest.mark.gpu
# new tokens and query heads of one key head: rows for each of the five widths that the two attention kernels work in
ROWS = [(1, 1), (12, 1), (7, 3), (8, 4), (14, 3)]


@pytest.mark.parametrize("H,n", ROWS)
@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
def test_attention_sums_of_q_keep_their_bits(ops, dtype, D, group, H, n):
    """Keys that are one number in all channels of a token: a score is that number times a sum of q, which two numbers of 8 bits do not
    hold.  The logarithm of a single weight is the score."""
    g = torch.Generator().manual_seed(D + group)
    part = torch.zeros(D)
    first = (D // group - 1) * group
    while True:       # numbers of 8 bits and three sizes: a sum of up to 24 bits, exact in 32
        size = torch.tensor([1.0, 2.0 ** -6, 2.0 ** -12])[torch.randint(0, 3, (group,), generator=g)]
        part[first:first + group] = torch.randint(128, 256, (group,), generator=g).float() / 4 * size * torch.where(torch.rand(group, generator=g) < 0.5, -1, 1)
        x = part.sum()
        rest = x - x.bfloat16().float()
        if abs(x) > 64 and abs(rest - rest.bfloat16().float()) > 2.0 ** -18.7 * abs(x):
            break
    want = float(part.double().sum())
    assert float(x) == want
    q = part.to(dtype)
    assert torch.equal(q.float(), part)
    q = (q.to(DEV) * torch.where(torch.arange(H, device=DEV) % 2 == 0, 1, -1).to(dtype)[:, None])[None, :, None].expand(1, H, n, D)
    for key in (1.0, -3.0):
        c = Filled(ops, gen(1), [n], 1, D, group, dtype, 16)
        # only the first key is in a row's sight, but for rows of later tokens: those keys are far lower
        c.k[:] = 0
        c.k[0, 0, 0] = key
        ops.kv4_append(c.data, c.k, c.v, c.slots, group)
        _, lse = ops.kv4_attention(q, c.data, c.table, c.len, group, None, 1.0, return_lse=True)
        score = want * key * torch.where(torch.arange(H, device=DEV) % 2 == 0, 1.0, -1.0).double()[None, :, None].expand(1, H, n)
        later = torch.arange(n, device=DEV).double().log()              # keys of zero: a score of 0 each
        exact = torch.logaddexp(score, later.expand_as(score))
        # two terms of 11 bits: 2^-22; their products' sum 2^-23 (cut off); factor, product with it, reference, sum with the logarithm and
        # change of its base 8 roundings of 2^-24; exponential and logarithm 2^-17 (as in `attention`)
        assert bool(((lse.double() - exact).abs() <= (2.0 ** -22 + 2.0 ** -23 + 2.0 ** -21) * score.abs() + 2.0 ** -17).all())
    ops.check_status()


def put_values(ops, c, v):
    """v [B, Hk, L, D] in the place of a filled cache's values."""
    c.v = v.to(c.dtype)
    ops.kv4_append(c.data, c.k, c.v, c.slots, c.group)


@pytest.mark.parametrize("H,n", ROWS)
@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, 1e13), (torch.bfloat16, -1e30), (torch.bfloat16, 1e-20), (torch.float16, 65504.0), (torch.float16, 6e-8)], **names)
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32)])
def test_attention_of_constant_values(ops, dtype, value, D, group, H, n):
    """Groups of one value have no step: the references take the value itself along."""
    g = gen(70)
    c = Filled(ops, g, [n, 500, 3000], 1, D, group, dtype, 64)
    put_values(ops, c, torch.full_like(c.v, value, dtype=torch.float32))
    got = check_attention(ops, randn(g, 3, H, n, D, dtype=dtype), c)
    assert bool((got == torch.tensor(value, dtype=dtype)).all())


@pytest.mark.parametrize("H,n", [(7, 1), (10, 3)])
@pytest.mark.parametrize("order", ["zeros first", "zeros last", "in turn"])
@pytest.mark.parametrize("value", [1e15, 1e30])
def test_attention_of_values_of_different_sizes(ops, value, order, H, n):
    """Rows of zeros before, behind and between large ones count as keys, within a warp, between warps and between blocks."""
    g = gen(71)
    lengths = [700, 40000, 90]
    c = Filled(ops, g, lengths, 1, 128, 64, torch.bfloat16, 64, k_scale=0.3)
    at = torch.arange(c.v.shape[2], device=DEV)[None, :]
    half = torch.tensor(lengths, device=DEV)[:, None] // 2
    zero = {"zeros first": at < half, "zeros last": at >= half, "in turn": at // 5 % 2 == 0}[order][:, None, :, None]
    for v in (torch.full_like(c.v, value, dtype=torch.float32), c.v.float() * value, torch.where(at[..., None, None].transpose(1, 2) % 2 == 0, value, 1e-20).expand_as(c.v)):
        put_values(ops, c, torch.where(zero, 0.0, v))
        check_attention(ops, randn(g, 3, H, n, 128, dtype=torch.bfloat16), c)


@pytest.mark.parametrize("H", [4, 12])
@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, 1e30), (torch.float16, 60000.0)], **names)
def test_attention_of_constant_values_over_a_long_context(ops, dtype, value, H):
    g = gen(72)
    c = Filled(ops, g, [131071], 1, 64, 32, dtype, 64)
    put_values(ops, c, torch.full_like(c.v, value, dtype=torch.float32))
    got = check_attention(ops, randn(g, 1, H, 2, 64, dtype=dtype), c)
    assert bool((got == torch.tensor(value, dtype=dtype)).all())


def test_cache_offsets_beyond_32_bits_within_a_page(ops):
    """One page of 2^24 tokens, 2.7 GB: rows at its start, on both sides of byte 2^31 and at its end, written, read and attended to."""
    D, group, page, g = 128, 32, 1 << 24, gen(73)
    data = torch.zeros_like(ops.kv4_empty(1, 1, page, D, group, DEV))
    slice_bytes = data.shape[3]
    border = (1 << 31) // slice_bytes * 16
    at = torch.cat([torch.arange(s, s + 16) for s in (0, border - 16, border, border + 16, page - 16)])[None]
    slots = at.to(torch.int32).to(DEV)
    q = randn(g, 1, 4, 1, D, dtype=torch.bfloat16)
    # keys in line with the queries' sum: what the other 2^24 tokens - zeros - count for stays small
    k = (2 * q.sum(1, keepdim=True).expand(1, 1, at.shape[1], D) + 0.1 * randn(g, 1, 1, at.shape[1], D)).to(torch.bfloat16)
    v = randn(g, 1, 1, at.shape[1], D, dtype=torch.bfloat16)
    ops.kv4_append(data, k, v, slots, group)
    for x, y in zip((k, v), ops.kv4_read(data, slots, D, group, torch.bfloat16)):
        want = stands_for(x, group)
        assert bool(((y.double() - want).abs() <= HALF[x.dtype] * 1.001 * want.abs() + TINY[x.dtype]).all())
    written = data.flatten(0, 2).any(-1).nonzero().flatten()                       # slices of 16 tokens
    assert written.tolist() == sorted({int(t) // 16 for t in at[0]})
    got = ops.kv4_attention(q, data, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([page], dtype=torch.int32, device=DEV), group)
    kk, vv = (stands_for(x, group)[0, 0] for x in (k, v))
    s = q[0, :, 0].double() @ kk.T * D ** -0.5
    top = s.amax(-1, keepdim=True).clamp(min=0)
    p = torch.exp(s - top)
    want = p @ vv / (p.sum(-1, keepdim=True) + (page - at.shape[1]) * torch.exp(-top))
    # bf16's half step, a weight's 2^-11 on codes of 15 steps at most, scores and the sum of 2^24 numbers to 2^-10
    assert bool(((got[0, :, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * vv.abs().amax()).all())
    ops.check_status()


def test_an_expired_wait_is_not_replaced_by_a_number_out_of_range(ops):
    """One status word a device: the code of a wait that ran out stays, whatever the calls behind it find."""
    from psa_b200 import _lib
    g = gen(74)
    c = Filled(ops, g, [64, 64], 1, 64, 32, torch.bfloat16, 16)
    word = ops.status_word(torch.device(DEV))
    one = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = torch.full((2, 1), 2 ** 30, dtype=torch.int32, device=DEV)
    row = randn(g, 2, 1, 1, 64, dtype=torch.bfloat16)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)

    def planned():
        ops.plan_pages(torch.full_like(c.table, -1), one * 0, one, one, none, 16, 1)
    calls = {"append": lambda: ops.kv4_append(c.data, row, row, bad, 32), "read": lambda: ops.kv4_read(c.data, bad, 64, 32, torch.bfloat16), "plan": planned,
             "plan in place": lambda: ops.plan_pages(c.table.clone(), c.len.clone(), one * 99, one, none.clone(), 16, 1), "length": lambda: ops.kv4_attention(row, c.data, c.table, c.len + 999, 32),
             "page": lambda: ops.kv4_attention(row, c.data, c.table + 10 ** 6, c.len, 32), "many rows": lambda: ops.kv4_attention(row.expand(2, 20, 1, 64), c.data, c.table + 10 ** 6, c.len, 32),
             "release": lambda: ops.release_pages(c.table, c.len.clone(), one.bool(), one[:1].clone(), one[:1].clone(), 16)}
    for name, call in calls.items():
        for before, text in ((0, "out of range"), (_lib.PSA_ERR_TIMEOUT, "wait expired")):
            word.fill_(before)
            call()
            with pytest.raises(RuntimeError, match=text):
                ops.check_status()
                pytest.fail(name)
    ops.check_status()


def test_attention_of_more_tokens_than_it_takes_is_refused(ops):
    c = Filled(ops, gen(75), [20], 1, 64, 32, torch.bfloat16, 16)
    with pytest.raises(ValueError, match="tokens"):
        ops.kv4_attention(torch.zeros(1, 1, 65536, 64, dtype=torch.bfloat16, device=DEV), c.data, c.table, c.len, 32)
    ops.check_status()


@pytest.mark.parametrize("dtype", [*TYPES, torch.float32], **names)
@pytest.mark.parametrize("layout", ["half", "pairs"])
def test_rotary_axes_in_forward_mode(ops, dtype, layout):
    """A tangent is turned as its operand is: of q, of k, of both, with a gradient wanted beside it, without gradients, of any layout."""
    from torch.autograd import forward_ad
    g = gen(76)
    pos = torch.randint(0, 999, (2, 2, 9), generator=g, device=DEV)
    ang = angles(pos, (12, 20), 1e4, False, 64)
    q, tq = (randn(g, 2, 9, 3, 64, dtype=dtype).transpose(1, 2) for _ in range(2))
    k, tk = randn(g, 2, 2, 9, 64, dtype=dtype), randn(g, 2, 1, 9, 1, dtype=dtype).expand(2, 2, 9, 64)
    plain = ops.rotate_axes(q, k, pos, (12, 20), layout=layout)

    def check(duals, tangents):
        outs = ops.rotate_axes(duals[0], duals[1], pos, (12, 20), layout=layout)
        for out, want, t in zip(outs, plain, tangents):
            primal, tangent = forward_ad.unpack_dual(out)
            assert torch.equal(primal, want) and (tangent is None) == (t is None)
            if t is not None:
                near_turned(tangent.detach(), t, ang, layout)
        return outs
    with forward_ad.dual_level():
        check((forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)), (tq, tk))
        check((forward_ad.make_dual(q, tq), k), (tq, None))
        check((q, forward_ad.make_dual(k, tk)), (None, tk))
        check((q, k), (None, None))
        with torch.no_grad():
            check((forward_ad.make_dual(q, tq), k), (tq, None))
        alone = forward_ad.unpack_dual(ops.rotate_axes(forward_ad.make_dual(q, tq), None, pos, (12, 20), layout=layout))
        near_turned(alone.tangent, tq, ang, layout)
        leaf = q.detach().clone().requires_grad_()
        outs = check((forward_ad.make_dual(leaf, tq), k), (tq, None))
        (back,) = torch.autograd.grad(forward_ad.unpack_dual(outs[0]).primal, leaf, tq)
        near_turned(back, tq, -ang, layout)
        # a tangent that comes to the gradient of the ordinary path is not dropped either
        leaf = q.detach().clone().requires_grad_()
        out = ops.rotate_axes(leaf, None, pos, (12, 20), layout=layout)
        try:
            (back,) = torch.autograd.grad(out, leaf, forward_ad.make_dual(q, tq))
        except RuntimeError as e:
            assert "jvp" in str(e)
        else:
            near_turned(forward_ad.unpack_dual(back).tangent, tq, -ang, layout)
    assert all(torch.equal(a, b) for a, b in zip(ops.rotate_axes(q, k, pos, (12, 20), layout=layout), plain))
    ops.check_status()


@pytest.mark.parametrize("requests,tokens", [(3, 20), (1100, 20), (3, 20000)])
@pytest.mark.parametrize("where", ["beside", "in place"])
def test_pages_of_no_slot_are_reported(ops, where, requests, tokens):
    """A request's page that is none, and one that the pool names: their tokens have no slot, and the status word says so."""
    def state(table_page, pool_page):
        width = tokens // 16 + 2
        table = torch.full((requests, width), -1, dtype=torch.int32, device=DEV)
        table[:, 0] = torch.arange(requests, device=DEV)
        table[1, 0] = table_page
        pool = torch.arange(requests, 2 * requests * width, dtype=torch.int32, device=DEV)
        pool[-1] = pool_page                             # the first page that is given away: request 0's
        return table, torch.full((requests,), 5, dtype=torch.int32, device=DEV), pool, torch.tensor([pool.numel()], dtype=torch.int32, device=DEV)

    def planned(*pages):
        table, lengths, pool, free = state(*pages)
        out = (table, lengths, free) if where == "in place" else None
        return ops.plan_pages(table, lengths, torch.full_like(lengths, tokens), pool, free, 16, tokens, out=out)[3]
    good = planned(1, 2 * requests * (tokens // 16 + 2))
    ops.check_status()
    assert bool((good >= 0).all())
    for pages in ((-1, 7), (1, -9), (2 ** 27, 7), (1, 2 ** 31 - 1)):
        slots = planned(*pages)
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status()
        gone = torch.zeros_like(slots, dtype=torch.bool)
        if pages[0] != 1:
            gone[1, :11] = True                          # places 5 .. 15 of its first page
        else:
            gone[0, 11:27] = True                        # its second page
        assert torch.equal(slots < 0, gone)
    ops.check_status()


@pytest.mark.parametrize("requests", [3, 70, 1500])
def test_release_puts_only_pages_into_the_pool(ops, requests):
    """Entries that are no page of any cache stay out of the pool, without a gap in it; lengths out of range end at 0 and are reported."""
    g = torch.Generator().manual_seed(requests)
    width, page = 70, 16
    table = torch.randperm(requests * width, generator=g).view(requests, width).to(torch.int32)
    lengths = torch.randint(0, width * page + 1, (requests,), generator=g).to(torch.int32)
    lengths[0] = width * page
    bad = torch.rand(requests, width, generator=g) < 0.1
    bad[1] = True
    bad[2] = False
    wrong = torch.tensor([-1, -2 ** 31, 2 ** 31 - 1, 2 ** 31 // page]).to(torch.int32)
    table[bad] = wrong[torch.arange(int(bad.sum())) % 4]
    which = torch.rand(requests, generator=g) < 0.7
    which[:3] = True
    room = requests * width + 5
    pool = torch.full((room,), -7, dtype=torch.int32)
    want = []
    for b in reversed(range(requests)):
        if which[b]:
            held = table[b, :-(-int(lengths[b]) // page)].tolist()
            want += [p for p in reversed(held) if 0 <= p < 2 ** 31 // page]
    state = [t.to(DEV) for t in (table, lengths, which, pool, torch.tensor([4], dtype=torch.int32))]
    ops.release_pages(*state, page)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert state[4].item() == 4 + len(want) and state[3][4:4 + len(want)].tolist() == want
    assert bool((state[3][:4] == -7).all())                       # what lies behind the free ones is nobody's
    assert torch.equal(state[1].cpu(), torch.where(which, 0, lengths)) and torch.equal(state[0].cpu(), table)
    # lengths out of range: nothing below zero, a whole row above its end
    far = torch.tensor([-5, width * page + 1, 3], dtype=torch.int32, device=DEV)
    rows = torch.arange(3 * width, dtype=torch.int32, device=DEV).view(3, width)
    pool, free = torch.full((3 * width,), -7, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.release_pages(rows, far, torch.ones(3, dtype=torch.bool, device=DEV), pool, free, page)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert far.tolist() == [0, 0, 0] and free.item() == 1 + width
    assert pool[:1 + width].tolist() == [2 * width] + list(reversed(range(width, 2 * width))) and bool((pool[1 + width:] == -7).all())
    ops.check_status()


@pytest.mark.parametrize("counts_dtype", [torch.int32, torch.int64], **names)
def test_refused_requests_answer_nothing(ops, counts_dtype):
    """Of three requests one fills its row and one finds the pool empty: `granted` says so on the device, their rows are zeros, the others'
    are as without them; in a captured step too."""
    from psa_b200.cache import KV4Cache, PageTable
    g = gen(77)
    B, H, D, n = 4, 4, 64, 3
    table = PageTable(B, 64, 9, 16, DEV)
    cache = KV4Cache(table, 1, D, torch.bfloat16)
    held = torch.tensor([20, 62, 48, 0], device=DEV)
    # pages: 2, 4 and 3 of 9; the first step needs none for request 0, one that the pool does not have for 2 and for 3, and 1's row is full
    rows = [randn(g, B, 1, 62, D, dtype=torch.bfloat16) for _ in range(2)]
    cache.append(*rows, table.reserve(held, 62))
    ops.check_status()
    want_counts = torch.tensor([n, 0, 0, 0], device=DEV)
    k, v = (randn(g, B, 1, n, D, dtype=torch.bfloat16) for _ in range(2))
    q = randn(g, B, H, n, D, dtype=torch.bfloat16)
    counts = torch.full((B,), n, dtype=counts_dtype, device=DEV)

    def step():
        slots = table.reserve(counts, n)
        ok = table.granted(counts, slots)
        cache.append(k, v, slots)
        return ok, cache.attend(q, ok)
    ok, out = step()
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert ok.dtype == torch.int32 and torch.equal(ok.long(), want_counts)
    assert table.lengths.tolist() == [23, 62, 48, 0] and not bool(out[1:].any()) and bool(out[0].any(-1).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok, out = step()
    graph.replay()
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    assert torch.equal(ok.long(), want_counts) and table.lengths.tolist() == [26, 62, 48, 0] and not bool(out[1:].any())
    table.release(torch.tensor([False, True, False, False], device=DEV))
    ok, out = step()
    ops.check_status()
    assert ok.tolist() == [n] * B and bool(out.any(-1).all()) and table.lengths.tolist() == [29, 3, 51, 3]


@pytest.mark.parametrize("dtype", TYPES, **names)
def test_calls_without_the_native_module(ops, monkeypatch, dtype):
    """Laid out in Python, every operator gives the same bits."""
    from psa_b200 import _lib
    from psa_b200.cache import KV4Cache, PageTable

    def everything():
        g = gen(78)
        table = PageTable(3, 200, 40, 16, DEV)
        cache = KV4Cache(table, 2, 64, dtype)
        got = []
        for n, counts in ((90, [90, 3, 0]), (1, [1, 1, 1]), (4, [4, 0, 3])):
            q, k, v = (randn(g, 3, n, h, 64, dtype=dtype).transpose(1, 2).requires_grad_() for h in (4, 2, 2))
            count = torch.tensor(counts, dtype=torch.int32, device=DEV)
            pos = (table.lengths[:, None] + torch.arange(n, dtype=torch.int32, device=DEV)).expand(3, 3, n)
            beside = ops.plan_pages(table.table, table.lengths, count, table.pool, table.free, 16, n)
            slots = table.reserve(count, n)
            turned = ops.rotate_axes(q, k, pos, (8, 12, 12))
            got += [*turned, *torch.autograd.grad(turned, (q, k), [torch.ones_like(t) for t in turned]), ops.rotate_axes(q.detach(), None, pos, (32, 0, 0), layout="pairs")]
            cache.append(turned[1].detach(), v.detach(), slots)
            got += [*beside, slots, cache.attend(turned[0].detach(), count), *cache.read(slots)]
            got += ops.kv4_attention(turned[0].detach(), cache.data, table.table, table.lengths, 32, count, 0.3, return_lse=True)
        ops.check_status()
        return got
    native = everything()
    monkeypatch.setattr(ops, "_calls", _lib.NoCalls)
    for a, b in zip(native, everything()):
        assert torch.equal(a, b) and a.stride() == b.stride()


@pytest.mark.parametrize("H", [2, 20])
def test_attention_of_the_longest_row_of_a_table(ops, H):
    """2^31 - 16 tokens, all on one page of 16: the number of tiles, and places beyond 2^30, fit their 32 bits; so do places of pages that are
    not there."""
    page, width = 16, (1 << 27) - 1
    data = ops.kv4_empty(1, 1, page, 64, 64, DEV)
    g = gen(79)
    row = randn(g, 1, 1, 1, 64, dtype=torch.bfloat16).expand(1, 1, page, 64)
    ops.kv4_append(data, row, row, torch.arange(page, device=DEV)[None], 64)
    q = randn(g, 1, H, 1, 64, dtype=torch.bfloat16)
    table = torch.zeros(1, width, dtype=torch.int32, device=DEV)
    length = torch.tensor([width * page], dtype=torch.int32, device=DEV)
    k = stands_for(row, 64)[0, 0, 0]
    score = (q[0, :, 0].double() @ k) / 8
    for tokens in (width * page, 1 << 30):
        table[0, tokens // page:] = -1
        out, lse = ops.kv4_attention(q, data, table, length, 64, return_lse=True)
        if tokens < width * page:
            with pytest.raises(RuntimeError, match="out of range"):
                ops.check_status()
        # a lane adds two weights a slice, of 2^27 slices in 148 x 2 blocks' 4 warps or more: 2^-24 of the sum each
        adds = 2 * 2 ** 27 / (148 * 2 * 4)
        assert bool(((lse[0, :, 0].double() - score - math.log(tokens)).abs() <= adds * 2.0 ** -24 + 2.0 ** -10).all())
        # every value is the same, so is every output: weights and their products with it are rounded alike but for what sums lose
        assert bool(((out[0, :, 0].double() - k).abs() <= 2.0 ** -8 * k.abs() + (2 * adds * 2.0 ** -24 + 2.0 ** -11) * 15 * k.abs().amax()).all())
    ops.check_status()


def test_numbers_beyond_32_bits_are_out_of_range(ops):
    """Slots and counts of 64 bits whose lower halves would do: skipped, refused or cut, and reported."""
    g = gen(80)
    far = 2 ** 32
    data = torch.zeros_like(ops.kv4_empty(1, 1, 16, 64, 32, DEV))
    row = randn(g, 1, 1, 3, 64, dtype=torch.bfloat16)

    def reported():
        with pytest.raises(RuntimeError, match="out of range"):
            ops.check_status()
    ops.kv4_append(data, row, row, torch.tensor([[far, far + 5, -far + 7]], device=DEV), 32)
    reported()
    assert not bool(data.any())
    ops.kv4_append(data, row, row, torch.tensor([[0, 1, 2]], device=DEV), 32)
    ops.check_status()
    assert not bool(ops.kv4_read(data, torch.tensor([[far, far + 1]], device=DEV), 64, 32, torch.bfloat16)[0].any())
    reported()
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([3], dtype=torch.int32, device=DEV)
    pool, free = torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    _, after, _, slots = ops.plan_pages(table, lengths, torch.tensor([far + 1], device=DEV), pool, free, 16, 2)
    reported()
    assert after.tolist() == [3] and slots.tolist() == [[-1, -1]]
    q = randn(g, 1, 2, 2, 64, dtype=torch.bfloat16)
    assert not bool(ops.kv4_attention(q, data, table, lengths, 32, torch.tensor([-far + 2], device=DEV)).any())
    reported()


@pytest.mark.parametrize("H,n", [(3, 2), (6, 2), (7, 3), (8, 4), (14, 3)])
@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, 1e9), (torch.bfloat16, 1e30), (torch.float16, 6e4)], **names)
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32)])
def test_attention_rows_do_not_feel_what_they_do_not_see(ops, dtype, value, D, group, H, n):
    """Large values of later tokens of the same call, random or constant: the rows before them keep every bit."""
    g = gen(81)
    lengths = [300, 64, 17]
    c = Filled(ops, g, lengths, 1, D, group, dtype, 16)
    c.v *= 2.0 ** -10
    ops.kv4_append(c.data, c.k, c.v, c.slots, group)
    q = randn(g, 3, H, n, D, dtype=dtype)
    clean = check_attention(ops, q, c)
    for big in (value * torch.rand(3, 1, 1, D, generator=g, device=DEV), torch.full((3, 1, 1, D), value, device=DEV)):
        v = c.v.clone()
        for b, length in enumerate(lengths):
            v[b, :, length - 1] = big[b, :, 0].to(dtype)
        keep, c.v = c.v, v
        ops.kv4_append(c.data, c.k, c.v, c.slots, group)
        got = check_attention(ops, q, c)
        c.v = keep
        assert torch.equal(got[:, :, :n - 1], clean[:, :, :n - 1])


@pytest.mark.parametrize("H,n", ROWS)
@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, 1e10), (torch.bfloat16, 1e30), (torch.float16, 6e4)], **names)
@pytest.mark.parametrize("D,group", [(64, 32), (128, 64)])
def test_attention_of_large_values_without_weight(ops, dtype, value, D, group, H, n):
    """Keys that point away from every query, with values far beyond the others': what they are worth is what their weight times their value
    is, and the others' codes keep their bits."""
    g = gen(82)
    c = Filled(ops, g, [900, 2000], 1, D, group, dtype, 64, k_scale=0.2)
    u = torch.sign(randn(g, D))
    q = (u + 0.3 * randn(g, 2, H, n, D)).to(dtype)
    away = torch.rand(2, 1, 2000, 1, generator=g, device=DEV) < 0.03
    away[:, :, -n:] = False
    c.v *= 2.0 ** -10
    size = {1e10: 20.0, 1e30: 40.0, 6e4: 20.0}[value] * 8 / D ** 0.5          # scores of some -8 size: 2^-230 and 2^-460
    c.k = torch.where(away, (-size * u).to(dtype), c.k)
    c.v = torch.where(away, (value * torch.rand(c.v.shape, generator=g, device=DEV)).to(dtype), c.v)
    ops.kv4_append(c.data, c.k, c.v, c.slots, group)
    check_attention(ops, q, c)


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
def test_cache_rounds_next_to_a_tie(ops, dtype, D, group):
    """Values and lowest values so near zero that the rest of a quotient lies next to a tie and is none: the nearer of the 16 values, where
    they meet exactly the even one."""
    tiny = [0.0, 2.0 ** -9, -2.0 ** -9, 2.0 ** -14, -2.0 ** -14, 2.0 ** -17, -2.0 ** -17, 2.0 ** -20, -2.0 ** -20, 2.0 ** -24, -2.0 ** -24]
    if dtype == torch.bfloat16:
        tiny += [2.0 ** -30, -2.0 ** -30]
    rows, codes = [], []
    for step in (1.0, 0.5, 3.0):
        for k in range(15):
            for x in tiny:                                      # (x - lowest) / step = k + 1/2 + x / step
                row = torch.full((group,), 7 * step)
                lowest = -(k + 0.5) * step
                row[0], row[1], row[2:] = lowest, lowest + 15 * step, x
                if bool((row.to(dtype).float() == row).all()):
                    rows.append(row)
                    codes.append(k + (1 if x > 0 or (x == 0 and k % 2) else 0))
            for low in tiny:                                    # lowest near zero, values at ties: (k + 1/2) step - lowest
                row = torch.full((group,), (k + 0.5) * step)
                row[0], row[1] = low, 15 * step
                if bool((row.to(dtype).float() == row).all()) and low < step / 2:
                    wide = (torch.tensor(15 * step, dtype=torch.float64) - low) / 15
                    if wide >= step and float(wide - step) < step * torch.finfo(dtype).eps / 2:          # cut off to the type: the step itself
                        rows.append(row)
                        codes.append(k + (1 if low < 0 or (low == 0 and k % 2) else 0))
    assert len(rows) > 300
    n, per = len(rows), D // group
    x = torch.stack(rows).to(dtype).to(DEV).repeat(1, per)[None, None]
    want = torch.tensor(codes, device=DEV)[:, None].expand(n, group).clone()
    data = ops.kv4_empty((n + 15) // 16, 1, 16, D, group, DEV)
    slots = torch.arange(n, device=DEV)[None]
    ops.kv4_append(data, x, x, slots, group)
    step, low, _ = scales(x, group)
    for y in ops.kv4_read(data, slots, D, group, dtype):
        z = y.double().unflatten(-1, (-1, group))
        got = torch.round((z - low) / step)[0, 0]                # the value it stands for is off by a rounding, far less than half a step
        for g in range(per):
            assert torch.equal(got[:, g, 2:].long(), want[:, 2:])


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
def test_cache_codes_of_values_of_many_sizes(ops, dtype, D, group):
    """Random values of sizes from 1 to 2^-20, whole numbers of a step among them, against quotients in 64 bits."""
    g = gen(83)
    n = 20000
    x = randn(g, 1, 2, n, D) * 2.0 ** -torch.randint(0, 21, (1, 2, n, D), generator=g, device=DEV)
    grid = torch.rand(1, 2, n, 1, generator=g, device=DEV) < 0.5
    x = torch.where(grid & (torch.rand(x.shape, generator=g, device=DEV) < 0.8), torch.round(x * 8) / 4, x).to(dtype)
    data = ops.kv4_empty(n // 16, 2, 16, D, group, DEV)
    slots = torch.randperm(n, generator=g, device=DEV)[None]
    ops.kv4_append(data, x, x.flip(-1), slots, group)
    for v, y in zip((x, x.flip(-1)), ops.kv4_read(data, slots, D, group, dtype)):
        want = stands_for(v, group)
        assert bool(((y.double() - want).abs() <= HALF[dtype] * 1.001 * want.abs() + TINY[dtype]).all())
    ops.check_status()


@pytest.mark.parametrize("dtype", TYPES, **names)
@pytest.mark.parametrize("D,group", SIZES)
def test_cache_steps_are_cut_off_exactly(ops, dtype, D, group):
    """A highest value that is 15 numbers of the type, and a lowest so little above zero that 32 bits do not see the difference: the step is the next
    smaller number, and lowest + 15 steps is not above the highest."""
    eps = torch.finfo(dtype).eps
    rows = []
    for step in (1.0, 3.0, 0.375, 1 + 8 * eps):
        for low in (0.0, 2.0 ** -24, 2.0 ** -23, -2.0 ** -24, 2.0 ** -14, -2.0 ** -14):
            row = torch.linspace(0, 15, group) * step
            row[0], row[1] = low, 15 * step
            row[2:] = row[2:].clamp(min=step / 4)
            if bool((row[:2].to(dtype).float() == row[:2]).all()):
                rows += [row, -row]
    if dtype == torch.float16:      # the sum of highest and 15 steps does not fit 24 bits
        for high, low in ((1023 * 2.0 ** -24, -1.0244140625), (2047 * 2.0 ** -24, -1.19921875)):
            row = torch.linspace(low, high, group)
            rows += [row, -row]
    x = torch.stack(rows).to(dtype).to(DEV).repeat(1, D // group)[None, None]
    n = x.shape[2]
    data = ops.kv4_empty((n + 15) // 16, 1, 16, D, group, DEV)
    slots = torch.arange(n, device=DEV)[None]
    ops.kv4_append(data, x, x, slots, group)
    want = stands_for(x, group)
    for y in ops.kv4_read(data, slots, D, group, dtype):
        assert bool(((y.double() - want).abs() <= HALF[dtype] * 1.001 * want.abs() + TINY[dtype]).all())
    step, low, _ = scales(x, group)
    assert bool((low + 15 * step <= x.double().unflatten(-1, (-1, group)).amax(-1, keepdim=True)).all())
