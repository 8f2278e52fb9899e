"""The waits of the 8-bit product, on the CPU: a warp whose lanes read the timer on either side of the limit has one
answer.  The two functions are taken from the kernels' source and compiled with 32 lanes in place of a warp."""
import os
import re
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tiny-kernel_b200", "csrc")

HARNESS = r"""
#include <cstdint>
#include <cstdio>
#define __device__
#define __forceinline__ inline
struct Fp8MatmulParams { unsigned* err; unsigned long long timeout_ns; };
constexpr unsigned kErrFp8Wait = 128u;
// the lane at work: it looks at the barrier `tries` times, and the timer says 1 at first and `now` from then on
static int complete_from, tries, reads;
static uint64_t now;
static bool any_lane;
static void atomicOr(unsigned* p, unsigned v) { *p |= v; }
static bool mbar_try_wait(uint64_t*, uint32_t) { return ++tries >= complete_from; }
static uint64_t global_timer_ns() { return reads++ == 0 ? 1 : now; }
static bool __any_sync(unsigned, bool) { return any_lane; }
%s
int main() {
  for (int early = 0; early <= 32; ++early) {  // lanes that read the timer just before the limit
    unsigned err = 0;
    bool dead[32] = {};
    any_lane = false;
    for (int lane = 0; lane < 32; ++lane) {
      Fp8MatmulParams p{&err, 1000};
      tries = reads = 0, complete_from = 64 * 2 + 3;  // complete just behind the second read
      now = lane < early ? 1001 : 1002;
      uint64_t bar = 0;
      wait_phase(&bar, 0, dead[lane], p);
      any_lane = any_lane || dead[lane];
    }
    const bool gave_up = dead[31];
    int answers = 0;
    for (int lane = 0; lane < 32; ++lane) answers += agreed(dead[lane]);
    printf("%%d %%d %%d %%u\n", early, (int)gave_up, answers, err);
  }
}
"""


def source():
    with open(os.path.join(CSRC, "tk_fp8_matmul.cu")) as f:
        return f.read()


def function(text, name):
    """The definition of a function, up to the brace that closes it."""
    start = re.search(r"^__device__ [^\n]*\b%s\(" % name, text, re.M).start()
    depth, at = 0, text.index("{", start)
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start:i + 1]


def test_lanes_that_wait_together_have_one_answer(tmp_path):
    code = HARNESS % (function(source(), "wait_phase") + "\n" + function(source(), "agreed"))
    (tmp_path / "wait.cpp").write_text(code)
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(tmp_path / "wait"), str(tmp_path / "wait.cpp")], check=True)
    lines = subprocess.run([str(tmp_path / "wait")], check=True, capture_output=True, text=True).stdout.split("\n")[:33]
    rows = [tuple(map(int, l.split())) for l in lines]
    assert [r[0] for r in rows] == list(range(33))
    assert all(answers in (0, 32) for _, _, answers, _ in rows)
    assert [answers for _, _, answers, _ in rows] == [32] * 32 + [0]  # one lane is enough
    assert all((err == 128) == (answers == 32) for _, _, answers, err in rows)


def test_every_wait_of_a_loop_is_agreed_on():
    """In the kernels each wait whose answer a whole warp acts on is followed by the warp's agreement."""
    text = source()
    acts = [m.start() for m in re.finditer(r"if \(dead\) break;\n\s+(?:const int n = |if \(elect_one|tcgen05_fence_after)", text)]
    assert len(acts) == 9  # copies, products and sums of three forms
    for at in acts:
        assert text[:at].rstrip().endswith("dead = agreed(dead);")
