"""CPU: what the operators around the causal attention of a prompt refuse, before anything reaches a GPU."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def ops():
    from psa_b200 import ops
    return ops


def x(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


POS = torch.zeros(3, 2, 5, dtype=torch.int64)


@pytest.mark.parametrize("q,k,positions,sections,more", [
    (x(2, 4, 5), None, POS, (16, 24, 24), {}),
    (x(2, 4, 5, 128), x(1, 4, 5, 128), POS, (16, 24, 24), {}),
    (x(2, 4, 5, 128), x(2, 4, 6, 128), POS, (16, 24, 24), {}),
    (x(2, 4, 5, 128), x(2, 4, 5, 128, dtype=torch.float16), POS, (16, 24, 24), {}),
    (x(2, 4, 5, 120), None, POS, (20, 20, 20), {}),
    (x(2, 4, 5, 272), None, POS, (36, 50, 50), {}),
    (x(2, 4, 5, 128), None, POS, (16, 24, 23), {}),
    (x(2, 4, 5, 128), None, POS, (64,), {}),
    (x(2, 4, 5, 128), None, POS, (-1, 40, 25), {}),
    (x(2, 4, 5, 128), None, POS[:, :, :4], (16, 24, 24), {}),
    (x(2, 4, 5, 128), None, torch.zeros(3, 3, 5, dtype=torch.int64), (16, 24, 24), {}),
    (x(2, 4, 5, 128), None, POS.float(), (16, 24, 24), {}),
    (x(2, 4, 5, 128), None, POS, (16, 24, 24), dict(layout="interleaved")),
    (x(2, 4, 5, 128), None, POS, (16, 24, 24), dict(theta=0.0)),
    (x(2, 4, 5, 128), None, POS, (16, 24, 24), dict(theta=float("nan"))),
    (x(2, 4, 5, 128), None, POS, (16, 24, 24), dict(inv_freq=[1.0] * 63)),
    (x(2, 4, 5, 128), None, POS, (16, 24, 24), dict(inv_freq=[float("inf")] * 64)),
    (x(2, 4, 5, 128, dtype=torch.float64), None, POS, (16, 24, 24), {}),
])
def test_rotate_axes_refuses(ops, q, k, positions, sections, more):
    with pytest.raises(ValueError):
        ops.rotate_axes(q, k, positions, sections, **more)


def test_there_is_no_cpu_path(ops):
    i = torch.zeros(2, dtype=torch.int32)
    data = ops.kv4_empty(2, 1, 16, 64, 32, "cpu")
    for call in (lambda: ops.rotate_axes(x(2, 4, 5, 128), None, POS, (16, 24, 24)),
                 lambda: ops.plan_pages(i.view(2, 1), i, i, i, i[:1], 16, 1),
                 lambda: ops.release_pages(i.view(2, 1), i, i.bool(), i, i[:1], 16),
                 lambda: ops.kv4_append(data, x(1, 1, 2, 64), x(1, 1, 2, 64), i[None], 32),
                 lambda: ops.kv4_read(data, i[None], 64, 32, torch.bfloat16),
                 lambda: ops.kv4_attention(x(2, 1, 1, 64), data, i.view(2, 1), i, 32)):
        with pytest.raises(RuntimeError):
            call()


def test_cache_refuses(ops):
    data, i = ops.kv4_empty(2, 2, 16, 64, 32, "cpu"), torch.zeros(1, 3, dtype=torch.int32)
    k = x(1, 2, 3, 64)
    bad = [
        lambda: ops.kv4_empty(2, 2, 24, 64, 32, "cpu"),
        lambda: ops.kv4_empty(0, 2, 16, 64, 32, "cpu"),
        lambda: ops.kv4_empty(2, 2, 16, 96, 32, "cpu"),
        lambda: ops.kv4_slice_bytes(64, 128),
        lambda: ops.kv4_slice_bytes(128, 16),
        lambda: ops.kv4_append(data, k.float(), k.float(), i, 32),
        lambda: ops.kv4_append(data, k, k[:, :, :2], i, 32),
        lambda: ops.kv4_append(data, k, k.half(), i, 32),
        lambda: ops.kv4_append(data, k[:, :1], k[:, :1], i, 32),
        lambda: ops.kv4_append(data, k, k, i, 64),
        lambda: ops.kv4_append(data.transpose(0, 1), k, k, i, 32),
        lambda: ops.kv4_append(data.char(), k, k, i, 32),
        lambda: ops.kv4_append(data, k[0], k[0], i, 32),
        lambda: ops.kv4_read(data, i[0], 64, 32, torch.bfloat16),
        lambda: ops.kv4_read(data, i, 64, 32, torch.float32),
        lambda: ops.kv4_attention(x(1, 3, 1, 64), data, i, i[0, :1], 32),
        lambda: ops.kv4_attention(x(1, 4, 1, 128), data, i, i[0, :1], 32),
        lambda: ops.kv4_attention(x(2, 4, 1, 64), data, i, i[0, :1], 32),
        lambda: ops.kv4_attention(x(1, 4, 1, 64), data, i[0], i[0, :1], 32),
        lambda: ops.kv4_attention(x(4, 1, 64), data, i, i[0, :1], 32),
        lambda: ops.kv4_attention(x(1, 4, 1, 64, dtype=torch.float32), data, i, i[0, :1], 32),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()


def test_pages_refuse(ops):
    from psa_b200.cache import PageTable
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: ops.plan_pages(i, i, i, i, i[:1], 16, 1),
                 lambda: ops.plan_pages(i.view(2, 2), i[:2], i[:2], i, i[:1], 24, 1),
                 lambda: ops.plan_pages(i.view(2, 2), i[:2], i[:2], i, i[:1], 16, 0),
                 lambda: ops.plan_pages(i.view(2, 2), i[:2], i[:2], i[:0], i[:1], 16, 1),
                 lambda: ops.release_pages(i.view(2, 2), i[:2], i[:2], i, i[:1], 16),
                 lambda: ops.release_pages(i.view(2, 2), i[:2], i[:3].bool(), i, i[:1], 16),
                 lambda: ops.release_pages(i.view(2, 2), i[:2], i[:2].bool(), i, i[:1], 8),
                 lambda: PageTable(0, 10, 10, 16, "cpu"), lambda: PageTable(1, 0, 10, 16, "cpu"), lambda: PageTable(1, 10, 0, 16, "cpu"),
                 lambda: PageTable(1, 10, 10, 20, "cpu")):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        PageTable(1, 10, 10, 16, "cpu")


# ---------------------------------------------------------------- the C entry points: numbers only, nothing is launched
P = 4096     # an aligned address that no refused call follows


def refused(rc, word):
    from psa_b200 import _lib
    assert rc in (_lib.PSA_ERR_ARG, _lib.PSA_ERR_UNSUPPORTED) and word in _lib.last_error(), (rc, _lib.last_error())


def test_rotate_axes_entry_refuses():
    from psa_b200._lib import lib

    def call(n=1, src=P, dst=2 * P, stride=64, heads=1, bits=64, axis=0, axes=1, batch=1, seq=1, dim=64, dtype=2, turns=True):
        i3 = (C.c_int64 * 6)(*[stride] * 6)
        return lib.psa_rotate_axes((C.c_void_p * 2)(src, src), i3, (C.c_void_p * 2)(dst, dst), i3, (C.c_int32 * 2)(heads, heads), n, P, bits,
                                   (C.c_int64 * 3)(), (C.c_uint64 * 256)() if turns else None, (C.c_uint8 * 256)(*[axis] * 256), axes, batch, seq, dim,
                                   1, 0, dtype, None)
    for kw, word in ((dict(n=3), "operands"), (dict(n=0), "operands"), (dict(src=P + 8), "aligned"), (dict(dst=P), "operand 0"), (dict(stride=60), "multiples"),
                     (dict(heads=0), "operand 0"), (dict(bits=16), "16 bits"), (dict(axis=1), "axis 1"), (dict(axes=9), "9 axes"), (dict(batch=0), "shape"),
                     (dict(seq=0), "shape"), (dict(dim=24), "head_dim"), (dict(dim=272), "head_dim"), (dict(dtype=7), "dtype"), (dict(turns=False), "null")):
        refused(call(**kw), word)


def test_pages_entries_refuse():
    from psa_b200._lib import lib

    def call(requests=2, width=4, pool=8, page=16, tokens=1, scratch=10 ** 6, table=P):
        return lib.psa_plan_pages(table, P, P, P, P, P, P, P, P, P, scratch, requests, width, pool, page, tokens, P, None)
    for kw in (dict(requests=0), dict(requests=65536), dict(width=0), dict(width=2 ** 28), dict(pool=0), dict(pool=2 ** 27), dict(page=8), dict(page=0),
               dict(tokens=0), dict(tokens=2 ** 30 + 1), dict(scratch=8), dict(table=None)):
        refused(call(**kw), "psa_plan_pages")

    def apart(**same):
        names = ("table", "lengths", "counts", "pool", "free", "table_out", "lengths_out", "free_out", "slots")
        at = {n: P * (i + 1) for i, n in enumerate(names)}
        at.update({a: at[b] for a, b in same.items()})
        return lib.psa_plan_pages(*[at[n] for n in names], P * 20, 10 ** 6, 2, 4, 8, 16, 2 ** 30 + 1, P * 21, None)
    refused(apart(table_out="table", lengths_out="lengths", free_out="free"), "tokens")          # in place: only the number of tokens is wrong
    for same in (dict(lengths_out="counts"), dict(table_out="pool"), dict(free_out="lengths"), dict(slots="table"), dict(free_out="counts")):
        refused(apart(**same), "another input")
    for same in (dict(lengths_out="free_out"), dict(slots="table_out")):
        refused(apart(**same), "two outputs")
    refused(lib.psa_release_pages(P, P, None, P, P, 2, 4, 8, 16, P, None), "null")
    refused(lib.psa_release_pages(P, P, P, P, P, 2, 4, 8, 17, P, None), "page size 17")
    assert lib.psa_plan_pages_scratch_bytes(0) == 0


def test_cache_entries_refuse():
    from psa_b200._lib import lib

    def strides(s=64):
        return (C.c_int64 * 6)(*[s] * 6)

    def append(fn=lib.psa_kv4_append, data=P, k=P, stride=64, pages=4, heads=2, page=16, batch=1, tokens=1, dim=64, group=32, dtype=2):
        if fn is lib.psa_kv4_append:
            return fn(data, k, P, strides(stride), P, pages, heads, page, batch, tokens, dim, group, dtype, P, None)
        return fn(data, k, P, strides(stride), P, pages, heads, page, batch, tokens, dim, group, dtype, P, None)
    for fn in (lib.psa_kv4_append, lib.psa_kv4_read):
        for kw, word in ((dict(data=None), "null"), (dict(k=P + 4), "aligned"), (dict(stride=4), "strides"), (dict(pages=2 ** 27), "pages"), (dict(pages=0), "pages"),
                         (dict(heads=0), "heads"), (dict(page=24), "pages"), (dict(batch=0), "shape"), (dict(tokens=2 ** 31), "shape"), (dict(dim=32), "head_dim"),
                         (dict(group=16), "group"), (dict(group=128), "group"), (dict(dtype=0), "f16/bf16")):
            refused(append(fn, **kw), word)

    def attend(q=P, stride=64, scratch=2 ** 40, pages=4, page=16, width=3, batch=1, tokens=1, heads=4, kv=2, dim=64, group=32, dtype=1):
        return lib.psa_kv4_attention(q, strides(stride), P, P, P, None, P, strides(stride), None, P, scratch, pages, page, width, batch, tokens, heads, kv,
                                     dim, group, 1.0, dtype, P, None)
    for kw, word in ((dict(q=None), "null"), (dict(q=P + 2), "aligned"), (dict(stride=12), "strides"), (dict(scratch=0), "scratch"), (dict(pages=0), "pages"),
                     (dict(page=40), "pages"), (dict(width=2 ** 28), "pages"), (dict(batch=0), "requests"), (dict(batch=65536), "requests"),
                     (dict(tokens=65536), "tokens"), (dict(heads=3), "heads"), (dict(kv=0), "heads"), (dict(dim=256), "head_dim"), (dict(group=48), "group"),
                     (dict(dtype=0), "f16/bf16")):
        refused(attend(**kw), word)
    assert lib.psa_kv4_slice_bytes(128, 32) == 16 * 160 and lib.psa_kv4_slice_bytes(128, 16) == 0
    assert lib.psa_kv4_attention_scratch_bytes(0, 1, 1, 1, 64) == 0


def test_calls_leave_what_is_out_of_the_ordinary_to_their_wrappers(ops):
    """CPU tensors, numbers that are none, wrong counts of arguments: None, and nothing is launched."""
    from psa_b200 import _calls
    i, data = torch.zeros(2, dtype=torch.int32), ops.kv4_empty(2, 1, 16, 64, 32, "cpu")
    turns, axis = ops._rotary_plan(64, (32,), 1e4, False, None)
    assert _calls.rotate(x(2, 1, 1, 64), None, i.view(1, 2), turns, axis, True, False, 1) is None
    assert _calls.rotate(3, None, i, turns, axis, True, False, 1) is None and _calls.rotate() is None
    assert _calls.plan_pages(i.view(2, 1), i, i, i, i[:1], 16, 1, None) is None and _calls.plan_pages(None) is None
    assert _calls.append(data, x(1, 1, 2, 64), x(1, 1, 2, 64), i[None], 32) is None and _calls.append(data, 1, 2, 3, 4) is None
    assert _calls.read(data, i[None], 64, 32, 2) is None and _calls.read(data, i[None], 64, 2 ** 70, None) is None
    assert _calls.attend(x(2, 1, 1, 64), data, i.view(2, 1), i, 32, None, None, False) is None and _calls.attend(*[None] * 8) is None
    with pytest.raises(TypeError):
        _calls.status("cuda", 0)


def test_rotary_plan_counts_turns_to_the_last_bit(ops):
    from fractions import Fraction
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459")
    turns, axis = ops._rotary_plan(64, (8, 12, 12), 1e4, True, None)
    assert list(axis) == [0] * 8 + [1] * 12 + [2] * 12
    assert turns[0] == turns[8] == turns[20] == round(2 ** 64 / two_pi)          # frequency 1 at the head of each axis
    turns, _ = ops._rotary_plan(64, (32,), 1e4, False, tuple([7.0] + [0.0] * 30 + [-1.0]))
    assert turns[0] == round(7 * 2 ** 64 / two_pi) - 2 ** 64 and turns[1] == 0 and turns[31] == 2 ** 64 - round(2 ** 64 / two_pi)
