"""The part of the selection (csrc/beam.cu) that finds the first of many candidates, compiled for the host: threads stand for the CTA's threads, and every barrier lets some warps go on long
before the others, so that an order which nothing enforces shows."""
import re
import subprocess
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "koboldcpp_b200" / "csrc" / "beam.cu"

HOST = r"""
#include <atomic>
#include <barrier>
#include <chrono>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <thread>
#include <vector>
#include <algorithm>
#define __device__
#define __forceinline__ inline
#define B200_BEAM_MAX 64
#define B200_BEAM_KEEP 128
using std::min;
using std::max;
constexpr int PICK_THREADS = 128, PICK_WARPS = PICK_THREADS / 32, LIST = 64;
constexpr float NEG_INF = -INFINITY;
struct { int x; } thread_local threadIdx;
static std::barrier<> *block;
static std::vector<std::unique_ptr<std::barrier<>>> warps;
static int late;  // the warp that goes on at once; the others come later
static void __syncthreads() {
    block->arrive_and_wait();
    if (threadIdx.x / 32 != late) std::this_thread::sleep_for(std::chrono::milliseconds(5));
}
static uint64_t lanes[PICK_THREADS];
template <typename T> T __shfl_xor_sync(unsigned, T x, int off) {
    auto &w = *warps[threadIdx.x / 32];
    memcpy(&lanes[threadIdx.x], &x, sizeof(T));
    w.arrive_and_wait();
    T r;
    memcpy(&r, &lanes[threadIdx.x ^ off], sizeof(T));
    w.arrive_and_wait();
    return r;
}
static int atomicAdd(int *p, int v) { return std::atomic_ref<int>(*p).fetch_add(v); }
static unsigned __float_as_uint(float f) { unsigned u; memcpy(&u, &f, 4); return u; }
static float __uint_as_float(unsigned u) { float f; memcpy(&f, &u, 4); return f; }
"""

MAIN = r"""
static PickShared sh;
int main(int argc, char **argv) {  // candidates, how many are kept, warp that is first behind barriers
    const int n = atoi(argv[1]), keep = atoi(argv[2]);
    late = atoi(argv[3]);
    std::vector<Cand> all;
    for (int i = 0; i < n; i++) all.push_back({(double)((i * 7919) % 50), i});
    std::vector<Cand> want = all;
    std::sort(want.begin(), want.end(), before);
    block = new std::barrier<>(PICK_THREADS);
    for (int w = 0; w < PICK_WARPS; w++) warps.push_back(std::make_unique<std::barrier<>>(32));
    std::vector<std::thread> threads;
    std::atomic<int> wrong{0};
    for (int t = 0; t < PICK_THREADS; t++) threads.emplace_back([&, t] {
        threadIdx.x = t;
        auto each = [&](auto &&f) { for (int i = t; i < n; i += PICK_THREADS) f(all[i]); };
        if (t == 0) for (int p = 0; p < 2; p++) sh.n[p] = 0;
        __syncthreads();
        for (int phase = 0; phase < 2; phase++) {  // as the kernel has them, one behind the other
            if (first_of(sh, phase, keep, -(double)INFINITY, each) != min(n, keep)) wrong++;
            if (t < min(n, keep) && (sh.best[t].score != want[t].score || sh.best[t].at != want[t].at)) wrong++;
            __syncthreads();
        }
    });
    for (auto &t : threads) t.join();
    printf("%d\n", (int)wrong);
    return wrong != 0;
}
"""


def part(text, begin, end):
    a = text.index(begin)
    return text[a:text.index(end, a)]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    text = SOURCE.read_text()
    found = part(text, "struct Cand {", "// The score of a logit of beam b.") + part(text, "template <typename F>\n__device__ __forceinline__ int first_of", "template <typename T, bool WIDE>\n__global__")
    assert not re.search(r"\basm\b", found)
    d = tmp_path_factory.mktemp("order")
    (d / "order.cpp").write_text(HOST + found + MAIN)
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", str(d / "order.cpp"), "-o", str(d / "order")], check=True)
    return d / "order"


@pytest.mark.parametrize("n,keep", [(0, 3), (1, 1), (5, 8), (40, 8), (64, 64), (65, 4), (300, 5)])
@pytest.mark.parametrize("first", [0, 1, 3])
def test_all_warps_see_the_same_candidates(program, n, keep, first):
    r = subprocess.run([str(program), str(n), str(keep), str(first)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, f"{r.stdout.strip()} threads had something else"


SCORE = r"""
int main() {
    int wrong = 0;
    auto expect = [&](float base, double ref, double norm, float x, float want) {
        sh.base[0] = base_of(base, false, (float)ref); sh.ref[0] = ref; sh.norm[0] = norm;
        const float got = (float)score_of(sh, 0, x);
        if (!(got == want)) { printf("base %g ref %g norm %g logit %g: %g, not %g\n", base, ref, norm, x, got, want); wrong++; }
    };
    const float inf = INFINITY;
    for (float base : {-2.5f, 0.0f, inf, -inf, 3.4028234e38f}) for (double ref : {0.0, 3.0, -7.0, (double)inf}) for (float x : {-INFINITY, -3.4028234e38f, -1.0f, 0.0f, 2.0f, 3.4028234e38f, INFINITY}) {
        if (x > ref) continue;  // (the reference is the largest logit, rounded up)
        const bool none = base == -inf || x == -INFINITY || (ref == inf && x < inf);
        expect(base, ref, 0.5, x, none ? -inf : (float)(x == INFINITY ? base - 0.5 : base + (((double)x - ref) - 0.5)));
    }
    if (base_of(NAN, false, 0.f) != -inf || base_of(1.f, false, -inf) != -inf || base_of(1.f, true, -inf) != 1.0 || base_of(-inf, true, 0.f) != -inf) wrong++;
    return wrong != 0;
}
"""


def test_scores_are_never_no_numbers(tmp_path):
    """Beams whose score is +inf beside logits of +inf: the other tokens are none.  (A candidate that is no number would have no rank, and leave a place that nobody writes.)"""
    text = SOURCE.read_text()
    (tmp_path / "score.cpp").write_text(HOST + part(text, "struct Cand {", "template <typename F>\n__device__ __forceinline__ int first_of") +
                                        "static PickShared sh;\n" + SCORE)
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", str(tmp_path / "score.cpp"), "-o", str(tmp_path / "score")], check=True)
    r = subprocess.run([str(tmp_path / "score")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
