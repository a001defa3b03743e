"""Tile products whose waits give up (a hang that should never be): what is in flight then has to end
before the CTAs of a pair leave. The rule for it (csrc/pair_drain.h) runs here on the CPU, against a model of
the stages' barriers, for every way in which the two CTAs can have stopped. And the word that tells of it
(``ffn.status``), over a stand-in for the library."""

import contextlib
import shutil
import subprocess
import types

import pytest
import torch

from cernels_b200 import ffn
from cernels_b200.build import CSRC

MODEL = r"""
#include <cstdio>
#include <initializer_list>
#include "pair_drain.h"
using namespace cernels;

struct Barrier {  // an mbarrier with one arrival a phase; parts: 1 the block's bytes of one CTA
  int pending = 1, parts = 0;
  long long phase = 0;
  void settle() { if (pending == 0 && parts == 0) { ++phase; pending = 1; } }
  void announce(int n) { parts += n; --pending; settle(); }
  void cancel(int n) { parts -= n; settle(); }
  void land() { --parts; settle(); }
};

// CTA 0 started `mine` blocks, CTA 1 `other`, the MMAs read `read`; of the blocks not read, bit i of `landed` says
// whether a part has landed before the drain (two bits a block).
bool holds(int stages, long long mine, long long other, long long read, unsigned landed) {
  Barrier bars[8];
  const long long most = mine > other ? mine : other;
  bool flying[64] = {};
  int n = 0;
  for (long long i = 0; i < most; ++i) {
    Barrier& b = bars[i % stages];
    if (i < mine) b.announce(2);
    for (int cta = 0; cta < 2; ++cta) {
      if (i >= (cta ? other : mine)) continue;
      if (i < read || (landed >> (2 * (i - read) + cta) & 1)) b.land();
      else flying[2 * (i - read) + cta] = true, ++n;
    }
    if (i < read && b.phase != i / stages + 1) return false;  // the model itself
  }
  // every stage with something in flight has to be waited for, and the wait has to end with its last part only
  for (long long i = drain_first(mine, other, stages); i < most; ++i) {
    Barrier& b = bars[i % stages];
    const Drain action = drain_action(i, mine, other);
    if (action == Drain::kAnnounce) b.announce(1);
    if (action == Drain::kCancel) b.cancel(1);
    for (int cta = 0; cta < 2; ++cta)
      if (i >= read && flying[2 * (i - read) + cta]) {
        if (b.phase != i / stages) return false;  // the wait would have ended before this part
        flying[2 * (i - read) + cta] = false;
        b.land(), --n;
      }
    if (b.phase != i / stages + 1) return false;  // the wait would never end
  }
  return n == 0;
}

int main() {
  long long cases = 0;
  for (int stages : {3, 4, 6, 8})
    for (long long read = 0; read <= 2 * stages + 1; ++read)
      for (long long mine = read; mine <= read + stages; ++mine)
        for (long long other = read; other <= read + stages; ++other)
          for (unsigned mask = 0; mask < 4096; mask += stages > 4 ? 7 : 1, ++cases)
            if (!holds(stages, mine, other, read, mask * 0x9e3779b1u >> (stages > 4 ? 0 : 20))) {
              std::printf("stages %d mine %lld other %lld read %lld mask %u\n", stages, mine, other, read, mask);
              return 1;
            }
  std::printf("%lld cases\n", cases);
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_every_load_in_flight_is_waited_for(tmp_path):
    source, program = tmp_path / "model.cpp", tmp_path / "model"
    source.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O2", "-I", str(CSRC), str(source), "-o", str(program)], check=True)
    run = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("device,index", [(None, 3), (0, 0), (2, 2), (torch.device("cuda"), 3), (torch.device("cuda", 0), 0),
                                          (torch.device("cuda:5"), 5), ("cuda", 3), ("cuda:1", 1)])
def test_status_reads_the_word_of_the_device_that_is_asked_for(monkeypatch, device, index):
    words, current, calls = {index: 2}, [3], []

    @contextlib.contextmanager
    def on(d):
        before, current[0] = current[0], d
        yield
        current[0] = before

    def read(code, stream):  # as the C entry: reads and clears the current device's word
        calls.append((current[0], stream))
        code._obj.value = words.pop(current[0], 0)
        return 0

    monkeypatch.setattr(ffn._lib, "load", lambda: types.SimpleNamespace(cernels_ffn_status=read))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=100 + d))
    assert ffn.status(device) == 2 and ffn.status(device) == 0
    assert calls == [(index, 100 + index)] * 2 and current == [3]


def test_status_refusals(monkeypatch):
    with pytest.raises(RuntimeError, match="cpu"):
        ffn.status("cpu")
    monkeypatch.setattr(ffn._lib, "load", lambda: types.SimpleNamespace(
        cernels_ffn_status=lambda code, stream: 4, cernels_error_string=lambda code: b"CUDA error"))
    monkeypatch.setattr(torch.cuda, "device", contextlib.nullcontext)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=0))
    with pytest.raises(RuntimeError, match="cernels_ffn_status"):  # an error of the call is not a status
        ffn.status(0)
