"""The way out of an expired wait in the 8-bit cache's attention, without a GPU: the ring's bookkeeping that the kernel
compiles (csrc/ring.cuh), against a model of mbarriers, and the switch that expires waits."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "mserve_b200" / "csrc"

# A barrier completes a phase when the load of its stage lands.  In the model a load lands only when it is waited for with
# the parity of the phase that it completes; a wait with the other parity returns at once, as that phase is over.
MODEL = r"""
#include <cstdio>
#include <vector>
#include "ring.cuh"
using mskv::RingPlace;

template <int S> struct Model {
  uint32_t done[S] = {};           // completed phases of a stage's barrier
  bool flying[S] = {};
  int refused = 0;                 // loads into a stage that still had one
  void load(int s) { refused += flying[s]; flying[s] = true; }
  bool wait(int s, uint32_t phase) {
    if ((done[s] & 1) != phase) return true;
    if (!flying[s]) return false;  // nothing would ever complete it: the wait runs out
    flying[s] = false;
    ++done[s];
    return true;
  }
  int in_flight() const { int n = 0; for (bool f : flying) n += f; return n; }
};

// A piece of n tiles after `turn` others, as the kernel takes it; the wait for tile `expires` runs out (-1: none).
// planted: the stages drained in their order with the current phase.
template <int S> int piece(Model<S>& m, uint32_t turn, int n, int expires, bool planted) {
  RingPlace<S> place(turn);
  for (int i = 0; i < S && i < n; ++i) m.load(place.stage_ahead(i));
  for (int i = 0; i < n; ++i) {
    if (place.stage != (int)((turn + i) % S) || place.phase != ((turn + i) / S & 1)) return 1;
    if (i == expires) {
      if (planted) { for (int k = 0; k < S; ++k) m.wait(k, place.phase); return 0; }
      return place.drain(i, n, [&](int s, uint32_t p) { return m.wait(s, p); }) ? 0 : 2;
    }
    if (!m.wait(place.stage, place.phase)) return 3;
    if (i + S < n) m.load(place.stage);
    place.advance();
  }
  return 0;
}

template <int S> int all(bool planted, int& left) {
  for (int first = 0; first < 3 * S; ++first)
    for (int n = 0; n < 4 * S + 2; ++n)
      for (int e = -1; e < n; ++e) {
        Model<S> m;
        if (const int rc = piece(m, 0, first, -1, false)) return rc;
        if (const int rc = piece(m, (uint32_t)first, n, e, planted)) return 10 + rc;
        left += m.in_flight();
        if (m.refused) return 20;
      }
  return 0;
}

int main() {
  int left = 0, planted = 0;
  if (const int rc = all<3>(false, left) | all<4>(false, left) | all<6>(false, left)) { printf("rc %d\n", rc); return 1; }
  all<3>(true, planted); all<4>(true, planted); all<6>(true, planted);
  printf("left %d planted %d\n", left, planted);
  return left != 0 || planted == 0;
}
"""


def test_drain_waits_for_every_load_in_flight(tmp_path):
    """Whatever tile's wait runs out, after whatever tiles: no load is left, and none is waited for in vain."""
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "a C++ compiler builds the package too"
    (tmp_path / "model.cpp").write_text(MODEL)
    subprocess.run([cxx, "-std=c++17", "-O1", "-x", "c++", f"-I{CSRC}", str(tmp_path / "model.cpp"), "-o", str(tmp_path / "model")],
                   check=True)
    r = subprocess.run([str(tmp_path / "model")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


def test_kernel_uses_the_ring(built_lib):
    """What is tested above is what the kernel runs: it keeps no stage or phase beside the ring's."""
    source = (CSRC / "kv8_attention.cu").read_text()
    assert "RingPlace<kStages> place(turn);" in source and "place.drain(0, left," in source
    assert "% kStages" not in source and "phase ^= 1" not in source and source.count("turn += n;") == 1


def test_expire_waits_is_a_switch(built_lib):
    from mserve_b200 import _lib
    lib = _lib.lib()
    assert lib.mskv_kv8_expire_waits(5) == 0
    try:
        assert lib.mskv_kv8_expire_waits(-1) == 1
        assert lib.mskv_kv8_expire_waits(0) == 1
    finally:
        assert lib.mskv_kv8_expire_waits(0) == 0


@pytest.fixture
def expire(built_lib):
    from mserve_b200 import _lib
    yield _lib.lib().mskv_kv8_expire_waits
    _lib.lib().mskv_kv8_expire_waits(0)


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,G,D,Q,lens,lists", [(1, 1, 4, 128, 1, [300], False),              # a CTA of its own
                                                  (2, 2, 7, 128, 1, [4000, 5], False),          # clusters
                                                  (3, 2, 16, 64, 2, [9000, 7, 0], False),       # parts of segments
                                                  (400, 2, 3, 64, 1, None, False),              # a line across segments
                                                  (5, 2, 7, 256, 1, [700] * 5, True)])
def test_expired_waits_end(expire, B, H, G, D, Q, lens, lists):
    """The first wait of every part of the work counts as expired: the call ends, says so, writes what it owes of its output and leaves
    nothing behind for the next one."""
    import torch
    from mserve_b200 import _lib, ops
    g = torch.Generator().manual_seed(B + D)
    if lens is None:
        lens = torch.randint(0, 60, (B,), generator=g).tolist()
        lens[7], lens[201] = 4000, 300
    dev = torch.device("cuda")
    width = max(lens) // 16 + 1
    pages = ops.kv8_pages(B * width, H, D)
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).to(dev)
    n = torch.tensor(lens, dtype=torch.int32, device=dev)
    x = torch.randn(2, B, H, max(lens), D, generator=g).to(torch.bfloat16).to(dev)
    ops.kv8_append(pages, table, x[0], x[1], tok0=torch.zeros_like(n), counts=n)
    q = torch.randn(B, H * G, Q, D, generator=g).to(torch.bfloat16).to(dev)
    kw = dict(lens=n, max_tokens=max(lens))
    if lists:
        kw["blocks"] = torch.arange(width, dtype=torch.int32, device=dev).view(1, 1, -1).expand(B, H, -1)
    out = torch.full_like(q, float("nan"))
    expire(1)
    for _ in range(3):
        ops.kv8_attention(q, pages, table, out=out, **kw)
        with pytest.raises(RuntimeError, match="time"):
            ops.check_status(dev)
        assert (out == 0).all()                     # nothing was taken, and every row is written
    expire(0)
    want = ops.kv8_attention(q, pages, table, **kw)
    ops.check_status(dev)
    assert torch.isfinite(want).all() and (want != 0).any()
    expire(1)
    ops.kv8_attention(q, pages, table, **kw)
    expire(0)
    assert ops.take_status(dev) == _lib.STATUS_TIMEOUT
    assert torch.equal(ops.kv8_attention(q, pages, table, **kw), want)
    ops.check_status(dev)
