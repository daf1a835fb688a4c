"""CPU: bookkeeping and host-side ends of the operators around the causal attention of a prompt."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "pyramid-sparse-attention_b200", "csrc")

RING = r"""
#include <cstdio>
#include "kv4_ring.h"
// A barrier as the hardware has it: armed and landed phases; a wait for a parity passes when the phase it stands in has the other one.
struct Barrier {
  int armed = 0, landed = 0;
  bool passes(unsigned parity) const { return (unsigned)(landed & 1) != parity; }
};
// `copied` tiles are copied, one barrier of N after the other, at most N ahead of what is waited for; `waited` are waited for (lengths of
// another moment).  Every copy still in flight must hold the wait at the end up, and nothing else may.
template <int N> int check(int copied, int waited) {
  Barrier bars[N];
  psa::Ring<N> ring = {0, 0};
  int done = 0;
  for (int i = 0; i < copied; ++i) {
    if (i - N >= waited) break;                      // the copier gives up: no one hands its barrier back
    Barrier& b = bars[ring.at];
    for (; done <= i - N; ++done) bars[done % N].landed++;
    if (ring.at != i % N || b.armed != b.landed) return 1;
    b.armed++;
    ring.advance();
    const auto same = psa::Ring<N>::after(i + 1);
    if (same.at != ring.at || same.phase != ring.phase) return 3;
  }
  for (int i = 0; i < N; ++i)
    for (;;) {
      const bool over = bars[i].armed == bars[i].landed;
      if (bars[i].passes(ring.last(i)) != over) return 2;
      if (over) break;
      bars[i].landed++;
    }
  return 0;
}
int main() {
  for (int copied = 0; copied < 40; ++copied)
    for (int waited = 0; waited < 40; ++waited) {
      int bad = check<2>(copied, waited) + check<3>(copied, waited) + check<4>(copied, waited) + check<5>(copied, waited) + check<6>(copied, waited);
      if (bad) { std::printf("%d copied, %d waited for\n", copied, waited); return 1; }
    }
}
"""


def test_blocks_wait_for_all_that_they_copied(tmp_path):
    """The copying side's ring says at the end which phase of each barrier was armed last, whatever the computing side waited for."""
    src = tmp_path / "ring.cpp"
    src.write_text(RING)
    exe = str(tmp_path / "ring")
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", f"-I{CSRC}", str(src), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout


@pytest.mark.parametrize("batch,tokens,heads,kv_heads", [(1, 1, 4, 8), (1, 1, 5, 2), (1, 2 ** 62, 4, 1), (65536, 1, 4, 4), (1, 65536, 4, 4), (1, 1, 4, 0), (0, 1, 4, 4)])
def test_scratch_of_refused_sizes_is_none(batch, tokens, heads, kv_heads):
    """A C caller asks for the scratch before it calls: numbers that the call refuses end neither the process (a division by zero) nor give bytes."""
    from psa_b200._lib import LIB_PATH
    code = (f"import ctypes as C; f = C.CDLL({LIB_PATH!r}).psa_kv4_attention_scratch_bytes; f.restype = C.c_size_t; "
            f"print(f(C.c_int64({batch}), C.c_int64({tokens}), {heads}, {kv_heads}, 128))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.split()[-1] == "0", (r.returncode, r.stdout, r.stderr)


def test_scratch_holds_the_parts():
    from psa_b200._lib import lib
    few, many = (lib.psa_kv4_attention_scratch_bytes(1, n, 4, 1, 128) for n in (1, 65535))
    assert 0 < few < many


def test_threads_make_one_status_word(monkeypatch):
    """Whoever comes first makes the word of a device; nobody is given, or stores, the address of another."""
    import threading
    import time
    from types import SimpleNamespace

    import torch

    from psa_b200 import ops
    made, stored, got, real = [], [], [], torch.zeros

    def zeros(*shape, dtype=None, device=None):
        time.sleep(0.05)
        made.append(real(*shape, dtype=dtype))
        return made[-1]
    monkeypatch.setattr(ops, "_STATUS", {})
    monkeypatch.setattr(ops, "_calls", SimpleNamespace(status=lambda index, address: stored.append((index, address))))
    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: SimpleNamespace(synchronize=lambda: None))
    start = threading.Barrier(4)

    def work():
        start.wait()
        got.append(ops.status_word("cuda:7"))
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and stored == [(7, made[0].data_ptr())] and all(w is made[0] for w in got) and len(got) == 4


def test_native_calls_of_other_versions_are_not_loaded(monkeypatch, tmp_path):
    """The module's name says what it was compiled against; without one of the running versions, and with one that does not load, importing
    warns and every call is laid out by its wrapper."""
    import torch

    from psa_b200 import _lib
    from psa_b200.calls_name import calls_name
    here = os.path.dirname(_lib.__file__)
    now = calls_name()
    assert torch.__version__ in now and os.path.exists(os.path.join(here, now)) and _lib._calls is not _lib.NoCalls
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert calls_name() != now
    with pytest.warns(RuntimeWarning, match="is not there"):
        assert _lib.load_calls(os.path.join(here, calls_name())) is _lib.NoCalls
    broken = tmp_path / "_calls-broken.so"
    broken.write_bytes(b"not a library")
    with pytest.warns(RuntimeWarning, match="does not load"):
        assert _lib.load_calls(str(broken)) is _lib.NoCalls
    names = [n for n in dir(_lib._calls) if not n.startswith("_")]
    assert sorted(names) == ["append", "attend", "plan_pages", "read", "rotate", "status"]
    assert all(getattr(_lib.NoCalls, n)(0, 0) is None for n in names)


def test_numbers_of_64_bits_keep_their_side_of_the_range():
    import torch

    from psa_b200 import ops
    far = torch.tensor([5, -1, 2 ** 32 + 5, -2 ** 32, 2 ** 31, -2 ** 31 - 1, 2 ** 62], dtype=torch.int64)
    got = ops._ints32("slots", far, (7,))
    assert got.dtype == torch.int32 and got.tolist() == [5, -1] + [2 ** 31 - 1, -2 ** 31] * 2 + [2 ** 31 - 1]
    strided = torch.arange(8, dtype=torch.int32)[::2]
    assert ops._ints32("counts", strided, (4,)).is_contiguous() and ops._ints32("counts", strided, (4,)).tolist() == [0, 2, 4, 6]


def test_derivatives_of_derivatives_in_either_mode(monkeypatch):
    """Around a stand-in for the kernel (twice its operand, and half of it on the way back): tangents of operands and of the gradients that come
    in, of one operand and not of the other."""
    import torch
    from torch.autograd import forward_ad

    from psa_b200 import ops
    monkeypatch.setattr(ops, "_rotate", lambda xs, positions, plan, half, inverse: tuple((0.5 if inverse else 2.0) * x for x in xs))
    q, k, pos = torch.randn(1, 2, 3, 16), torch.randn(1, 1, 3, 16), torch.zeros(1, 3, dtype=torch.int64)
    tq, tk, gq, gk = torch.randn_like(q), torch.randn_like(k), torch.randn_like(q), torch.randn_like(k)
    with forward_ad.dual_level():
        for of_q, of_k in ((True, True), (True, False), (False, True), (False, False)):
            a, b = q.clone().requires_grad_(), k.clone().requires_grad_()
            x, y = ops.rotate_axes(forward_ad.make_dual(a, tq) if of_q else a, forward_ad.make_dual(b, tk) if of_k else b, pos, (8,))
            for out, t, has in ((x, tq, of_q), (y, tk, of_k)):
                tangent = forward_ad.unpack_dual(out).tangent
                assert torch.equal(tangent, 2 * t) if has else tangent is None
            for in_q in (True, False):
                up = forward_ad.make_dual(gq, tq) if in_q else gq
                da, db = torch.autograd.grad((x, y), (a, b), (up, gk), retain_graph=True)
                assert torch.equal(forward_ad.unpack_dual(da).primal, gq / 2) and torch.equal(db, gk / 2)
                tangent = forward_ad.unpack_dual(da).tangent
                assert torch.equal(tangent, tq / 2) if in_q else tangent is None
