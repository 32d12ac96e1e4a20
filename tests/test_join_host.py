"""The exchange between blocks that share a tile (csrc/mkx_join.h), run on the host: threads stand for the warps of a
block, and one of them is late on its way to every word that it reads, or leaves."""
import shutil
import subprocess

import pytest

from conftest import ROOT

SOURCE = r"""
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <mutex>
#include <thread>
#include <vector>
#include "mkx_join.h"

constexpr int WARPS = 8;
#ifndef GONE
#define GONE 99  // the warp that leaves: none
#define LIMIT_MS 20000
#else
#define LIMIT_MS 10
#endif
struct Barrier {
  std::mutex m;
  std::condition_variable cv;
  int come = 0, phase = 0;
  bool wait() {
    std::unique_lock<std::mutex> l(m);
    const int now = phase;
    if (++come == WARPS) {
      come = 0;
      ++phase;
      cv.notify_all();
      return true;
    }
    return cv.wait_for(l, std::chrono::milliseconds(LIMIT_MS), [&] { return phase != now; });
  }
};
struct Team {
  Barrier* barrier;
  int warp, late;
  bool ok = true;
  bool leads() const { return warp == 0; }
  bool meet() { return ok = barrier->wait(); }
  bool read(const int* w) const {
    if (warp == late) std::this_thread::sleep_for(std::chrono::milliseconds(4));
    return __atomic_load_n(w, __ATOMIC_SEQ_CST) != 0;
  }
  void write(int* w, bool v) const { __atomic_store_n(w, (int)v, __ATOMIC_SEQ_CST); }
  unsigned held(const unsigned* t) const { return __atomic_load_n(t, __ATOMIC_SEQ_CST); }
  unsigned take(unsigned* t) const { return __atomic_fetch_add(t, 1u, __ATOMIC_SEQ_CST); }
  void clear(unsigned* t) const { __atomic_store_n(t, 0u, __ATOMIC_SEQ_CST); }
};
#ifdef ONE_WORD
struct Words { union { int last; int others; }; };
#else
using Words = mkxa::JoinWords;
#endif

// Question 0: last_of, 1: others_done, of two parts each, of which the other one has delivered or not.
int main() {
  int wrong = 0;
  for (int code = 0; code < 64; ++code)
    for (int late : {1, 7}) {
      const int kind[3] = {code & 1, code >> 1 & 1, code >> 2 & 1};
      const unsigned there[3] = {(unsigned)(code >> 3 & 1), (unsigned)(code >> 4 & 1), (unsigned)(code >> 5 & 1)};
      unsigned tickets[3] = {there[0], there[1], there[2]};
      Words words{};
      Barrier barrier;
      std::vector<std::thread> warps;
      int bad[WARPS] = {};
      for (int w = 0; w < WARPS; ++w)
        warps.emplace_back([&, w] {
          Team team{&barrier, w, late};
          if (w == GONE) return;  // before the first question
          for (int i = 0; i < 3; ++i) {
            const bool yes = kind[i] ? mkxa::others_done(team, &tickets[i], 2, words) : mkxa::last_of(team, &tickets[i], 2, words);
            if (GONE < WARPS) {  // nobody hears yes, and everybody learns that somebody is missing
              bad[w] += yes || team.ok;
              return;
            }
            bad[w] += yes != (there[i] == 1);
          }
        });
      for (auto& t : warps) t.join();
      for (int b : bad) wrong += b;
      for (int i = 0; i < 3 && GONE >= WARPS; ++i) wrong += tickets[i] != (there[i] ? 0u : kind[i] ? 0u : 1u);
    }
  printf("%d\n", wrong);
  return 0;
}
"""


def _wrong(tmp_path, *flags):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ missing")
    (tmp_path / "join.cpp").write_text(SOURCE)
    subprocess.run([gxx, "-std=c++17", "-O1", "-pthread", *flags, "-I", str(ROOT / "reki_megakernel_b200" / "csrc"),
                    str(tmp_path / "join.cpp"), "-o", str(tmp_path / "join")], check=True)
    return int(subprocess.run([str(tmp_path / "join")], capture_output=True, text=True, timeout=120, check=True).stdout)


def test_every_warp_hears_the_same_answer(tmp_path):
    """All sequences of three questions, whichever of them are answered yes: a late warp reads the answer to its own."""
    assert _wrong(tmp_path) == 0


def test_one_word_for_both_questions_is_not_enough(tmp_path):
    """The same with both answers in one word: others_done writes before its first meeting, while a late warp still reads
    last_of's answer. (Shows that the test above sees it.)"""
    assert _wrong(tmp_path, "-DONE_WORD") > 0


@pytest.mark.parametrize("gone", [0, 5])
def test_a_warp_that_left_is_not_waited_for(gone, tmp_path):
    """A warp gave up before the first question (the one that asks, or another): the others come back within their limit,
    with a no, and know that the answer is none."""
    assert _wrong(tmp_path, f"-DGONE={gone}") == 0


def test_no_unbounded_barrier_among_warps_that_may_leave():
    """In the kernel of chunks a warp may leave its role early; between the roles' start and their common end nothing but
    mbarriers with a limit is waited for."""
    text = (ROOT / "reki_megakernel_b200" / "csrc" / "mk_attend.cu").read_text()
    body = text[text.index("chunk_kernel(const __grid_constant__"):text.index("// ---- host ---")]
    roles = body[body.index("if (warp >= 8) {"):body.rindex("__syncthreads();")]
    assert "__syncthreads" not in roles and "bar.sync" not in roles and "BarrierTeam" not in roles and "row_barrier" not in roles
    assert "BoundedTeam" in roles
