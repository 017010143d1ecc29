"""The ranks of the operators' stable sort do not rest on the order in which a warp's lanes run.

csrc/op_sort.cuh's `SortWalk` is compiled for the host.  The 32 lanes are coroutines that run one after the other from one warp-wide operation (vote, shuffle, barrier) to the next, in
ascending, descending and shuffled order: all that CUDA promises about lanes between two such operations.  Ranks have to be those of a stable sort in every order.
"""
import os
import shutil
import subprocess

import pytest

from helpers import ROOT

CUDA = next((d for d in (os.environ.get("CUDA_HOME"), "/usr/local/cuda") if d and os.path.exists(os.path.join(d, "include", "cuda_runtime.h"))), None)
SOURCE = r"""
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#undef __launch_bounds__
#define __launch_bounds__(...)
#undef __global__
#define __global__
#undef __shared__
#define __shared__
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>
#include <ucontext.h>
using std::min;

// ---- a warp: lanes run from one warp-wide operation to the next
static ucontext_t g_main, g_lane[32];
static int g_current, g_kind[32], g_arg[32];
static unsigned g_value[32], g_got[32];
static bool g_done[32];
enum { VOTE, SHUFFLE, BARRIER, END };
static unsigned meet(int kind, unsigned value, int arg) {
    const int me = g_current;
    g_kind[me] = kind, g_value[me] = value, g_arg[me] = arg;
    swapcontext(&g_lane[me], &g_main);
    return g_got[me];
}
static unsigned __ballot_sync(unsigned, int p) { return meet(VOTE, p != 0, 0); }
template <typename V> static V __shfl_sync(unsigned, V v, int from) { return (V)meet(SHUFFLE, (unsigned)v, from); }
static void __syncwarp(unsigned = 0xffffffffu) { meet(BARRIER, 0, 0); }
static int atomicAdd(int* p, int v) { const int old = *p; *p += v; return old; }
static int __popc(unsigned v) { return __builtin_popcount(v); }
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }
// not used by what is tested
template <typename V> static V __shfl_xor_sync(unsigned, V v, int) { abort(); return v; }
template <typename V> static V __shfl_up_sync(unsigned, V v, int) { abort(); return v; }
static void __syncthreads() { abort(); }
static float __uint_as_float(unsigned v) { float f; memcpy(&f, &v, 4); return f; }
static struct { struct { operator unsigned() const { return (unsigned)g_current; } } x; } g_thread;
static struct { unsigned x; } g_block, gridDim;
#define threadIdx g_thread
#define blockIdx g_block
#include "op_sort.cuh"

struct Source {
    const int* keys;
    int operator()(int64_t i) const { return keys[i]; }
    int id(int64_t i) const { return (int)i; }
    int key(int v) const { return v; }
};
static const std::vector<int>* g_keys;
static SortPlan g_plan;
static int* g_count;
static std::vector<int> g_rank;
static int g_steps_at_once;
template <int S> static void lane_body() {
    const Source source{g_keys->data()};
    SortWalk<Source, S> w(source, (int64_t)g_keys->size(), g_plan);
    for (int s0 = 0; s0 < g_plan.steps; s0 += S) {
        w.load(s0);
        w.add(g_count);
        for (int s = 0; s < S; ++s)
            if (s0 + s < g_plan.steps && (size_t)((s0 + s) * 32 + w.lane) < g_keys->size()) g_rank[(s0 + s) * 32 + w.lane] = w.rank[s];
    }
    g_done[g_current] = true;
    meet(END, 0, 0);
}
static void lane_main() { g_steps_at_once == 4 ? lane_body<4>() : lane_body<8>(); }

static bool run(int order, std::mt19937& rng) {
    static std::vector<char> stacks(32 * 65536);
    for (int l = 0; l < 32; ++l) {
        getcontext(&g_lane[l]);
        g_lane[l].uc_stack.ss_sp = stacks.data() + l * 65536;
        g_lane[l].uc_stack.ss_size = 65536;
        g_lane[l].uc_link = &g_main;
        makecontext(&g_lane[l], lane_main, 0);
        g_done[l] = false;
    }
    for (;;) {
        int lanes[32];
        for (int l = 0; l < 32; ++l) lanes[l] = order == 1 ? 31 - l : l;
        if (order == 2) std::shuffle(lanes, lanes + 32, rng);
        for (int l : lanes) g_current = l, swapcontext(&g_main, &g_lane[l]);
        for (int l = 1; l < 32; ++l)
            if (g_kind[l] != g_kind[0]) { printf("lanes meet in different operations\n"); return false; }
        if (g_kind[0] == END) return true;
        unsigned vote = 0;
        for (int l = 0; l < 32; ++l) vote |= g_value[l] << l;
        for (int l = 0; l < 32; ++l) g_got[l] = g_kind[0] == VOTE ? vote : g_kind[0] == SHUFFLE ? g_value[g_arg[l] & 31] : 0;
    }
}

int main() {
    std::mt19937 rng(5);
    for (int keys : {1, 2, 9, 33, 256, 1024})
        for (int entries : {1, 31, 100, 256, 257, 500, 1024})
            for (int skew : {0, 1})
                for (int order : {0, 1, 2}) {
                    std::vector<int> key(entries);
                    for (int& k : key) k = skew && rng() % 2 ? 0 : (int)(rng() % (keys + 1)) - 1;  // -1: no choice
                    const int steps = (entries + 31) / 32;
                    g_keys = &key;
                    g_plan = SortPlan();
                    g_plan.blocks = 1, g_plan.keys = keys, g_plan.align = 1, g_plan.steps = steps;
                    for (g_plan.bits = 0; 1 << g_plan.bits < keys; ++g_plan.bits) {}
                    std::vector<int> count(keys, 7), want(keys, 7);
                    g_count = count.data();
                    g_rank.assign(entries, -1);
                    g_steps_at_once = steps <= 4 ? 4 : 8;
                    if (!run(order, rng)) return 1;
                    for (int i = 0; i < entries; ++i)
                        if (key[i] >= 0 && g_rank[i] != want[key[i]]++) {
                            printf("%d entries of %d keys, lanes in order %d: entry %d has rank %d, not %d\n", entries, keys, order, i, g_rank[i], want[key[i]] - 1);
                            return 1;
                        }
                    if (count != want) { printf("counts\n"); return 1; }
                }
    return 0;
}
"""


@pytest.mark.skipif(CUDA is None or shutil.which("g++") is None, reason="needs g++ and the CUDA headers")
def test_ranks_do_not_depend_on_the_lanes_order(tmp_path):
    source, program = tmp_path / "warp.cpp", str(tmp_path / "warp")
    source.write_text(SOURCE)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-I", os.path.join(CUDA, "include"), "-I", os.path.join(ROOT, "tatara_b200", "csrc"), str(source), "-o", program], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
