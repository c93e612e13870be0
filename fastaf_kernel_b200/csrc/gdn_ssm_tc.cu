// gdn_ssm_tc.cu -- chunked (64 tokens) selective scan on the 5th-generation tensor cores:
// tcgen05.mma with TMEM accumulators, TMA-fed tiles, warp-specialised.
//
// With la_i the running sum of the log decays a inside a chunk and S the state in front of
// it (formulas in gdn_ssm_common.cuh), the chunk's 64 tokens are
//
//   y_i   = exp(la_i) S C_i + sum_{j <= i} M_ij x_j + D x_i,
//   M_ij  = (C_i . B_j) exp(la_i - la_j) dt'_j
//   S    <- exp(la_63) S + sum_j w_j x_j B_j^T,   w_j = exp(la_63 - la_j) dt'_j
//
// One CTA carries 128 state rows of one sequence through its chunks: one head of 128, or two
// heads of 64 of one group (they share B, C and the product C B^T).  State rows are the
// tensor core's M = 128, tokens its N, so the fp32 state [row][128] stays in TMEM columns
// [0, 128) for the whole sequence and the outputs come out transposed, [row][token].
// Products per chunk:
//   G    = C B^T                 scores [i][j]; A is the C tile's 64 rows (the other 64 rows
//                                of the M = 128 tile read what lies behind it and are unused)
//   Yi^T = bf16(S) C^T           the state's part, scaled by exp(la_i) per column afterwards
//   Ya^T = x^T bf16(M)^T         the chunk's own part
//   S   += (w x)^T B             w x in fp32, cut into three bf16 numbers (8 of its 24 bits each, so
//                                exactly), three products: the fp32 state is as good as fp32 sums
//                                (relative error 3e-7; two terms left 4e-6).  Terms one and two are
//                                a TMEM operand, which keeps 48 KB a chunk out of the shared
//                                memory's bandwidth.  The third has no TMEM columns of its own: with
//                                one head it lies in shared memory, where M leaves room; with two
//                                it takes the place of bf16(S) when Yi has read that; the local
//                                pass, which has neither M nor Yi, holds all three in TMEM.
// M's exponentials factor by blocks of 8 columns: exp(la_i - la_j) = exp(la_i - la_r)
// exp(la_r - la_j) with r the block's last column, both at most 1 for the rows below the
// block; the 8 rows of the block itself take one exponential per element.  So a row of 32
// columns takes 12 exponentials, and none overflows however strong the decays are.
//
// D x is added in fp32 where the outputs are formed, from the staged x tile.  On M's diagonal,
// where it needs no read of x, it is rounded to bf16 together with the token's own score: D to 8
// bits, an error of one sign for all tokens of a head, and own scores below half a step of D lost.
//
// Roles (28 warps), handing chunks to each other through mbarriers:
//   warp 0        issues the state update(c), then G(c + 1) (with two heads the update's third term
//                 behind that); allocates TMEM
//   warp 3        issues Yi(c), Ya(c) (one thread alone could not keep the tensor pipe busy)
//   warp 18       copies (TMA): three stages of C, B and x, two of z, and boxes further ahead
//                 into L2
//   warp 2        the chunk's gates
//   warps 4-7     state path: S -> bf16 copy (TMEM operand of Yi) and the decay of S
//   warps 12-15, 24-27   the terms of w x, 16 state rows each; the rows behind the last token set
//                 to zero
//   warps 16, 17, 1   M, a 32 x 32 block each
//   warps 8-11, 20-23   outputs, 32 tokens each: Yi, Ya from TMEM as accumulator fragments, D x,
//                 the gate z, transposed into bf16 rows in shared memory (stmatrix)
//   warp 19       output rows to global memory (TMA; the last, partial chunk by hand)
// The loops are kept rolled and the waits out of line: together they have to fit the SM's
// instruction caches (with everything unrolled a chunk took 7,200 cycles, two thirds of the
// issue slots waiting for instructions).
//
// What bounds it.  A chunk of one head takes about 2,500 cycles (1.35 us alone on its SM), of which
// the tensor pipe works 1,400 and HBM less; 16 x 8192 tokens, 32 heads of 128 in 16 groups: 1.0 ms,
// 3.3 TB/s, 324 TFLOP/s (the 512 chains are 3.5 waves of 148 CTAs, run as four).  No unit is full:
// every product waits for a role to turn accumulators into operands, and each hand-over (TMEM
// load, conversion, store, fence, barrier, issue) costs 400 to 700 cycles.  Pairs take 3,800: three
// warps form both heads' M in 2,500, and G has one buffer to wait for them.  With z a chunk of
// one head takes 3,300: its 16 K hardware exponentials and reciprocals alone are 1,024.
// What fp32 precision costs at 16 x 8192 (865 us in a graph, 735 without either): the third term's
// products 45 us, its way through shared memory 24, cutting w x in three instead of two about 30,
// D x in the epilogue 30.
// Measured and not kept: a third issuing warp or 30 warps (64 registers: spills, twice the time),
// M's scores 16 columns at a time with the diagonal block apart (4 x 2048 tokens in pairs with z,
// 71 -> 75 us), three stages of z in place of two (16 x 2048 tokens, 283 -> 278 us with z, 205
// -> 212 without).
//
// Every wait is bounded as in gdn_prefill_tc.cu: one that gives up records its site in the
// device status word and raises a shared flag, every role stops at its next wait, the
// issuing threads wait (bounded) for their own MMAs and copies, and the CTA frees TMEM.
#include <cuda_bf16.h>
#include <cstring>

#include "gdn_mma_sync.cuh"
#include "gdn_ssm_common.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace gdn {

namespace {

using namespace sm100;
using msync::ldsm_x4_t;
using msync::stsm_x4_t;

constexpr int kL = 64;              // tokens of a chunk
constexpr int kThreads = 896;
constexpr int kRows = 128;          // state rows of a CTA
constexpr int kStages = 3;          // of C, B, x
constexpr int kGateStages = 4;
constexpr int kPrefetch = 6;        // chunks the L2 prefetch runs ahead
constexpr int kZBehind = 2;         // chunks z's copies run behind the others
constexpr int kMWarps = 3, kYWarps = 8;
constexpr int kSplitWarps = 8, kUpdateWarps = 12;     // of the split; of the state path and the split

// Shared memory (bytes from the 1024-aligned base).  Tiles are 64 rows of 64 bf16 (one
// 128-byte swizzled atom, 8 KB), two atoms side by side.
constexpr uint32_t kTile = 16 * 1024;
constexpr uint32_t OFF_STAGE = 0;                                // kStages x [C | B | x]
constexpr uint32_t STAGE = 3 * kTile;
constexpr uint32_t ST_C = 0, ST_B = kTile, ST_X = 2 * kTile;
constexpr uint32_t OFF_M = OFF_STAGE + kStages * STAGE;          // 2 x [head][i][j], K-major, 8 KB each
constexpr uint32_t OFF_W3 = OFF_M + kTile;                       // one head: third term of w x, [token][row] as x
constexpr uint32_t OFF_Y = OFF_M + 2 * kTile;                        // 2 x z, then the output rows in its place
constexpr uint32_t OFF_GATE = OFF_Y + 2 * kTile;                 // kGateStages x 2 heads x Gates
constexpr uint32_t GATE = 1408;
constexpr uint32_t SMEM_BYTES = OFF_GATE + kGateStages * 2 * GATE;
static_assert(SMEM_BYTES <= 227 * 1024 - 1024, "shared memory map");

struct alignas(16) Gates {
    float la[64];         // log2 of the decays' products from the start of the chunk
    float lb[64];         // la_j - log2(dt'_j): 2^(la_i - lb_j) = exp(la_i - la_j) dt'_j
    float cf[64];         // exp(la_r - la_j) dt'_j, r = j | 7
    float e[64];          // exp(la_i)
    // w_j = exp(la_63 - la_j) dt'_j, pairs of tokens with equal (j / 2) % 4 side by side: what one
    // lane of a fragment needs (rows of 80 bytes: four lanes' reads in different banks)
    float w[4][20];
    float total;          // exp(la_63)
    float D;              // the skip term's, for the outputs
};
static_assert(sizeof(Gates) <= GATE, "gate block");

// TMEM columns (all 512 allocated).  One head: two buffers of G, so that the scores of a chunk
// need not wait for M of the one before; two heads: one, since Ya takes 64 columns per head
// (rows 0..63 use the first head's, rows 64..127 the second's).
template <bool PAIR>
struct Tm {
    static constexpr uint32_t S = 0;                         // [0, 128) fp32 state
    static constexpr uint32_t SB = 128;                      // [128, 192) bf16x2 copy of it
    static constexpr uint32_t G = 192;                       // lanes 0..63, 64 columns a buffer
    static constexpr int kG = PAIR ? 1 : 2;
    static constexpr uint32_t YI = G + 64 * kG, YA = YI + 64;
    static constexpr uint32_t W = YA + (PAIR ? 128 : 64);    // bf16x2 w x: 32 columns a term, two terms
    static constexpr uint32_t W3 = SB;                       // the third, with two heads
    static_assert(W + 64 == 512, "TMEM map");
    static constexpr uint32_t WL = 128;                      // local pass: three terms, two buffers
};

enum WaitSite { kSsmTma = 41, kSsmZ = 42, kSsmGates = 43, kSsmG = 44, kSsmM = 45, kSsmS = 46,
                kSsmMX = 48, kSsmUpdate = 47, kSsmCS = 53, kSsmIssue = 49, kSsmY = 50, kSsmStage = 51, kSsmFree = 52,
                kSsmRead = 54, kSsmThird = 55 };
constexpr uint64_t kDrainNs = 2000000000ull;
constexpr uint32_t kMaxSuspendNs = 1000000;

// Sequences may be cut into segments of `segment` tokens (a multiple of 64; as many as there
// are, without cuts) that run side by side.  Segment j of sequence n has slot
// cu_seqlens[n] / segment + n + j, so that the slots of different sequences are distinct
// whatever their lengths; a first pass (LOCAL) leaves in `ends` what every segment but a
// sequence's last adds to the state and in `decays` its decay, ssm_combine_kernel turns `ends` into the states behind the segments, and the main
// pass starts every segment from the one in front of it.
struct TcArgs {
    SsmArgs a;
    int slabs, per_group;    // CTAs per segment, per group
    uint64_t wait_ns;
    int64_t segment;
    float *ends;             // [slot][slab][128][128]
    float *decays;           // [slot][slab][128], one per state row
};

// The tokens of sequence n, clamped to [0, T].
__device__ __forceinline__ void sequence_of(const SsmArgs &p, int64_t n, int64_t &s0, int64_t &s1) {
    s0 = p.cu_seqlens[n];
    s1 = p.cu_seqlens[n + 1];
    s0 = s0 < 0 ? 0 : (s0 > p.rows ? p.rows : s0);
    s1 = s1 < s0 ? s0 : (s1 > p.rows ? p.rows : s1);
}
__device__ __forceinline__ int64_t first_slot(const TcArgs &a, int64_t n) {
    int64_t s0 = a.a.cu_seqlens[n];
    s0 = s0 < 0 ? 0 : (s0 > a.a.rows ? a.a.rows : s0);
    return s0 / a.segment + n;
}
__device__ __forceinline__ int64_t segments_of(const TcArgs &a, int64_t tokens) {
    return tokens > 0 ? (tokens + a.segment - 1) / a.segment : 1;
}

struct Bars {
    uint64_t full[kStages], empty[kStages], gates[kGateStages], ydone[kGateStages];
    uint64_t zfull[2], yst[2], yfree[2], mx[2], mready[2], update[2], last[2], g[2], mread[2];
    uint64_t s, cs, yread, third;
};

// What a wait looks at besides its barrier, at the end of the dynamic shared memory.
struct WaitControl {
    uint64_t limit;
    uint32_t hint, units;       // the limit, at most kMaxSuspendNs, and in units of wait_clock()
    int *status;
    volatile int abort;
};
// A clock of one register: units of 1024 ns.
__device__ __forceinline__ uint32_t wait_clock() { return static_cast<uint32_t>(global_timer_ns() >> 10); }
__device__ __forceinline__ WaitControl *wait_control() {
    extern __shared__ __align__(1024) uint8_t sm[];
    return reinterpret_cast<WaitControl *>(sm + SMEM_BYTES);
}

// A wait behind its first probe, out of line (see above).  `key` is the phase's parity and,
// above it, the WaitSite.
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t key) {
    WaitControl *ctl = wait_control();
    const uint64_t t0 = global_timer_ns(), limit = ctl->limit;
    const uint32_t hint = ctl->hint;
    for (;;) {
        if (mbar_try_wait_hint(bar, key & 1, hint)) return true;
        if (ctl->abort) return false;
        if (global_timer_ns() - t0 > limit) {
            if (ctl->status) atomicCAS(ctl->status, 0, static_cast<int>(key >> 1));
            ctl->abort = 1;
            return false;
        }
    }
}
// The same without suspending the thread: a suspended wait ends late, but not early, so that
// this one, for the first copies, is what notices a limit of a microsecond or less.
__device__ __noinline__ bool wait_polled(uint32_t bar, uint32_t key) {
    WaitControl *ctl = wait_control();
    const uint64_t t0 = global_timer_ns();
    while (!mbar_test_wait(bar, key & 1)) {
        if (ctl->abort) return false;
        if (global_timer_ns() - t0 > ctl->limit) {
            if (ctl->status) atomicCAS(ctl->status, 0, static_cast<int>(key >> 1));
            ctl->abort = 1;
            return false;
        }
    }
    return true;
}
// This CTA's own copies and MMAs, also after a give-up.
__device__ __noinline__ void wait_own(uint32_t bar, uint32_t key) {
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait_hint(bar, key & 1, kMaxSuspendNs)) {
        if (global_timer_ns() - t0 > kDrainNs) {
            WaitControl *ctl = wait_control();
            if (ctl->status) atomicCAS(ctl->status, 0, static_cast<int>(key >> 1));
            return;
        }
    }
}

// A barrier's phases are told apart by parity, so a wait for phase k (0, 1, ...) may only
// look while phase k + 1 cannot be complete; tests/test_ssm_chain_protocol.py models it.
struct Waiter {
    static __device__ __forceinline__ uint32_t key(uint32_t phase, int site) { return (phase & 1u) | (site << 1); }
    // The whole warp; it stays converged for the next .aligned tcgen05 instruction.
    __device__ __forceinline__ bool warp(uint32_t bar, uint32_t phase, int site) const {
        bool ok = mbar_try_wait(bar, phase & 1);
        if (!__all_sync(0xffffffffu, ok)) {
            if (!ok) ok = wait_slow(bar, key(phase, site));
            if (!__all_sync(0xffffffffu, ok)) return false;
        }
        tc_fence_after();
        return true;
    }
    // The same with no call in it: for a wait across which a warp keeps many registers.
    __device__ __forceinline__ bool warp_inline(uint32_t bar, uint32_t phase, int site) const {
        bool ok = mbar_try_wait(bar, phase & 1);
        if (!__all_sync(0xffffffffu, ok)) {
            WaitControl *ctl = wait_control();
            const uint32_t t0 = wait_clock();
            while (!ok && !ctl->abort) {
                ok = mbar_try_wait_hint(bar, phase & 1, ctl->hint);
                if (!ok && wait_clock() - t0 > ctl->units) {
                    if (ctl->status) atomicCAS(ctl->status, 0, site);
                    ctl->abort = 1;
                    break;
                }
            }
            if (!__all_sync(0xffffffffu, ok)) return false;
        }
        tc_fence_after();
        return true;
    }
    __device__ __forceinline__ void drain(uint32_t bar, uint32_t phase, int site) const {
        wait_own(bar, key(phase, site));
    }
};

__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger of the two, or NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ uint64_t bits2(uint32_t lo, uint32_t hi) {
    return f2(__uint_as_float(lo), __uint_as_float(hi));
}
// The leading 8 bits of two numbers as a pair of bf16 (cut off, not rounded), and what is left of
// them, exactly.
__device__ __forceinline__ uint32_t cut_bf2(uint64_t &v) {
    float a, b;
    unf2(v, a, b);
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    v = sub_f2(v, bits2(ua & 0xffff0000u, ub & 0xffff0000u));
    return __byte_perm(ua, ub, 0x7632);
}
// softplus(x) = max(x, 0) + log(1 + u), u = exp(-|x|) in (0, 1], with the logarithm from the
// series log(1 + u) = 2 (s + s^3/3 + s^5/5 + ...), s = u / (2 + u) <= 1/3, whose first term
// left out is below 2^-22 of the sum: a few instructions, and accurate relative to small
// results too.  (torch's softplus is x itself above 20, which this rounds to as well.)
__device__ __forceinline__ float softplus_series(float x) {
    const float u = ex2(-1.4426950408889634f * fabsf(x));
    const float s = __fdividef(u, 2.0f + u), q = s * s;
    float v = fmaf(q, 1.0f / 11.0f, 1.0f / 9.0f);
    v = fmaf(q, v, 1.0f / 7.0f);
    v = fmaf(q, v, 1.0f / 5.0f);
    v = fmaf(q, v, 1.0f / 3.0f);
    v = fmaf(q * v, s, s);
    return fmaxf(x, 0.0f) + 2.0f * v;
}

// PAIR: two heads of 64 rows; else one head of 128.  LOCAL: the state update alone (see TcArgs),
// from a segment's last chunk to its first: a token's weight, its decay to the segment's end, is
// then known when it comes, so the products accumulate without a pass over the state in between
// (0.75 us a chunk; in order, with the state decayed chunk by chunk, 0.2 more).  The scaled x has
// two places; its barriers are those of G.  A pair's gates take two warps (with one, 1 x 16,384
// tokens in 32 chains of pairs took 13 us more).
template <bool PAIR, bool LOCAL>
__global__ void __launch_bounds__(kThreads, 1)
ssm_tc_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap bmap,
              const __grid_constant__ CUtensorMap cmap, const __grid_constant__ CUtensorMap zmap,
              const __grid_constant__ CUtensorMap ymap, const TcArgs args) {
    extern __shared__ __align__(1024) uint8_t sm[];
    __shared__ Bars bars;
    __shared__ uint32_t tmem_slot;
    using TM = Tm<PAIR>;
    const SsmArgs &p = args.a;
    constexpr int kHeads = PAIR ? 2 : 1;
    constexpr int kGateReaders = LOCAL ? kUpdateWarps : kYWarps;    // the last to read a chunk's gates
    constexpr int kGateWriters = LOCAL && PAIR ? 2 : 1;             // warps that take the gates' turns
    constexpr int kUpdateArrivals = LOCAL ? kSplitWarps : kUpdateWarps;

    // (warp-uniform for the compiler too, so that the MMA warp's loop and descriptors are)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t lane_base = static_cast<uint32_t>(warp & 3) * 32;
    const int row = static_cast<int>(lane_base) + lane;    // this thread's TMEM lane
    const int64_t slot = blockIdx.x / args.slabs;
    int64_t n = slot;
    if (args.ends != nullptr) {
        // the last sequence whose first slot is not behind this one
        int64_t lo = 0, hi = p.num_seqs - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) >> 1;
            if (first_slot(args, mid) <= slot) lo = mid;
            else hi = mid - 1;
        }
        n = lo;
    }
    const int slab = static_cast<int>(blockIdx.x % args.slabs);
    const int g = slab / args.per_group, R = p.heads / p.groups;
    const int h0 = g * R + (slab % args.per_group) * kHeads;
    const bool lone = PAIR && (slab % args.per_group) * 2 + 1 >= R;   // a pair's second head is missing
    // (there are at least as many slots as sequences)
    if (!LOCAL && tid == 0 && slab == 0 && slot < p.num_seqs)
        check_seq_bounds(p.cu_seqlens, slot, p.num_seqs, p.rows, p.status);
    int64_t s0, s1;
    sequence_of(p, n, s0, s1);
    const int64_t segments = args.ends ? segments_of(args, s1 - s0) : 1, seg = args.ends ? slot - first_slot(args, n) : 0;
    const bool last = seg == segments - 1;
    if (seg < 0 || seg >= segments || (LOCAL && last)) return;      // (no such segment, or none needed)
    s0 += seg * args.segment;
    s1 = last ? s1 : s0 + args.segment;
    const int tokens = static_cast<int>(s1 - s0), nch = (tokens + kL - 1) / kL;
    const bool gated = !LOCAL && p.z != nullptr;
    const uint32_t sbase = smem_u32(sm);
    auto bar = [&](const uint64_t &b) { return smem_u32(&b); };
    const Waiter wait;

    // this thread's state row: of head h0, or for the second half of a pair of head h0 + 1
    const int hrow = PAIR ? (warp & 2) >> 1 : 0;
    // the slab's 128 state rows, one after the other in memory (64 for a lone head)
    const int64_t state_at = (n * p.heads + h0) * p.head_size * static_cast<int64_t>(kSsmState);
    const int64_t end_at = (slot * args.slabs + slab) * kRows;      // their place in the segments' workspace
    // the slab's columns in the rows of x, z and y (a lone head's twice: the copy is not stored)
    const int xc0 = h0 * p.head_size, xc1 = lone ? xc0 : xc0 + 64;

    if (nch == 0) {
        // An empty sequence keeps its state (or starts at zero).
        const int vecs = (lone ? 64 : kRows) * kSsmState / 4;
        for (int i = tid; i < vecs; i += kThreads)
            reinterpret_cast<float4 *>(p.new_state + state_at)[i] =
                p.state ? reinterpret_cast<const float4 *>(p.state + state_at)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    // where the state starts from, and its lines on their way into L2 meanwhile
    const float *const first = LOCAL      ? nullptr
                               : seg == 0 ? (p.state ? p.state + state_at : nullptr)
                                          : args.ends + (end_at - static_cast<int64_t>(args.slabs) * kRows) * kSsmState;
    if (first && tid < (lone ? 64 : kRows) * kSsmState / 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(first + tid * 32));
    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < kStages; ++i) {
                mbar_init(bar(bars.full[i]), 1);
                mbar_init(bar(bars.empty[i]), 2);
            }
            for (int i = 0; i < kGateStages; ++i) {
                mbar_init(bar(bars.gates[i]), kGateWriters);
                mbar_init(bar(bars.ydone[i]), kGateReaders);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar(bars.zfull[i]), 1);
                mbar_init(bar(bars.yst[i]), kYWarps);
                mbar_init(bar(bars.yfree[i]), 1);
                mbar_init(bar(bars.mx[i]), 1);
                mbar_init(bar(bars.mready[i]), kMWarps);
                mbar_init(bar(bars.update[i]), kUpdateArrivals);
                mbar_init(bar(bars.last[i]), 1);
                mbar_init(bar(bars.g[i]), 1);
                mbar_init(bar(bars.mread[i]), kMWarps);
            }
            mbar_init(bar(bars.s), 1);
            mbar_init(bar(bars.cs), 1);
            mbar_init(bar(bars.yread), kYWarps);
            mbar_init(smem_u32(&bars.third), kSplitWarps);
            WaitControl *ctl = wait_control();
            ctl->limit = args.wait_ns;
            ctl->hint = args.wait_ns < kMaxSuspendNs ? static_cast<uint32_t>(args.wait_ns) : kMaxSuspendNs;
            ctl->units = args.wait_ns >> 41 ? 0x7fffffffu : static_cast<uint32_t>(args.wait_ns >> 10);
            ctl->status = p.status;
            ctl->abort = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    // M's upper right blocks stay zero
    for (int i = tid; i < static_cast<int>(kHeads * kTile / 16); i += kThreads)
        reinterpret_cast<uint4 *>(sm + OFF_M)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_slot;
    auto gates_of = [&](int c, int head) -> Gates * {
        return reinterpret_cast<Gates *>(sm + OFF_GATE + ((c & (kGateStages - 1)) * 2 + head) * GATE);
    };
    auto gates_full = [&](int c) { return wait.warp(bar(bars.gates[c & (kGateStages - 1)]), c / kGateStages, kSsmGates); };

    if (warp == 0) {
        // -------------------------------------------------------------- state update and G
        // The whole warp runs the loop, so that its control flow and the descriptors stay
        // uniform; one elected lane issues.
        const uint64_t dC = smem_desc_sw128(sbase + OFF_STAGE + ST_C, 16, 1024);      // K-major
        const uint64_t dBk = smem_desc_sw128(sbase + OFF_STAGE + ST_B, 16, 1024);     // K-major
        const uint64_t dBm = smem_desc_sw128(sbase + OFF_STAGE + ST_B, 8192, 1024);   // MN-major
        constexpr int kAtom = 8192 >> 4, kStep = 2048 >> 4, kSt = STAGE >> 4;
        constexpr uint32_t id_g = idesc_bf16_f32(128, 64, false, false);
        constexpr uint32_t id_s = idesc_bf16_f32(128, 128, false, true), id_w3 = idesc_bf16_f32(128, 128, true, true);
        constexpr int kW3 = (OFF_W3 - OFF_STAGE - ST_B) >> 4;
        int ng = 0, ns = 0;
        auto scores = [&](int c) -> bool {      // G(c)
            const uint32_t st = (c % kStages) * kSt;
            if (!wait.warp(bar(bars.full[c % kStages]), c / kStages, kSsmTma)) return false;
            if (c >= TM::kG && !wait.warp(bar(bars.mread[c & (TM::kG - 1)]), c / TM::kG - 1, kSsmM)) return false;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    mma_ss(tm + TM::G + (c & (TM::kG - 1)) * 64, dC + st + (k >> 2) * kAtom + 2 * (k & 3), dBk + st + (k >> 2) * kAtom + 2 * (k & 3),
                           id_g, k > 0);
                mma_commit(bar(bars.g[c & (TM::kG - 1)]));
            }
            __syncwarp();
            ++ng;
            return true;
        };
        bool ok = __all_sync(0xffffffffu, wait_polled(bar(bars.full[0]), Waiter::key(0, kSsmTma)));
        if (!LOCAL && ok) ok = scores(0);
#pragma unroll 1
        for (int c = 0; ok && c < nch; ++c) {
            const uint32_t st = (c % kStages) * kSt;
            if (LOCAL && !(ok = wait.warp(bar(bars.full[c % kStages]), c / kStages, kSsmTma))) break;
            // (the split's warps and, but for the local pass, the state path's)
            if (!(ok = wait.warp(bar(bars.update[c & 1]), c >> 1, kSsmUpdate))) break;
            if (elect_one()) {                  // S += (w x)^T B: one term after the other against the same B
                const uint32_t w = tm + (LOCAL ? TM::WL + (c & 1) * 96 : TM::W);
#pragma unroll 4
                for (int k = 0; k < (LOCAL ? 12 : 8); ++k)
                    mma_ts(tm + TM::S, w + 8 * k, dBm + st + (k & 3) * kStep, id_s, !LOCAL || c > 0 || k > 0);
                if (!LOCAL && !PAIR) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_ss(tm + TM::S, dBm + kW3 + k * kStep, dBm + st + k * kStep, id_w3, 1);
                }
                if (LOCAL || !PAIR) {
                    mma_commit(bar(LOCAL ? bars.g[c & 1] : bars.s));
                    mma_commit(bar(bars.empty[c % kStages]));
                    if (LOCAL) mma_commit(bar(bars.empty[c % kStages]));   // (for the other issuing warp)
                }
            }
            __syncwarp();
            if (LOCAL || !PAIR) ++ns;
            if (!LOCAL && c + 1 < nch && !(ok = scores(c + 1))) break;
            if (!LOCAL && PAIR) {
                if (!(ok = wait.warp(smem_u32(&bars.third), c, kSsmThird))) break;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_ts(tm + TM::S, tm + TM::W3 + 8 * k, dBm + st + k * kStep, id_s, 1);
                    mma_commit(bar(bars.s));
                    mma_commit(bar(bars.empty[c % kStages]));
                }
                __syncwarp();
                ++ns;
            }
        }
        // No MMA or barrier arrive is in flight when the CTA leaves (after a give-up some may
        // have gone out without a commit of their own).
        if (elect_one()) mma_commit(bar(bars.last[0]));
        __syncwarp();
        wait.drain(bar(bars.last[0]), 0, kSsmIssue);
#pragma unroll 1
        for (int c = ng > TM::kG ? ng - TM::kG : 0; c < ng; ++c)
            wait.drain(bar(bars.g[c & (TM::kG - 1)]), c / TM::kG, kSsmG);
        if (LOCAL) {
#pragma unroll 1
            for (int c = ns > 2 ? ns - 2 : 0; c < ns; ++c) wait.drain(bar(bars.g[c & 1]), c >> 1, kSsmS);
        } else if (ns) {
            wait.drain(bar(bars.s), ns - 1, kSsmS);
        }
        __syncwarp();
    } else if (!LOCAL && warp == 3) {
        // -------------------------------------------------------------- Yi and Ya
        const uint64_t dC = smem_desc_sw128(sbase + OFF_STAGE + ST_C, 16, 1024);      // K-major
        const uint64_t dX = smem_desc_sw128(sbase + OFF_STAGE + ST_X, 8192, 1024);    // MN-major
        const uint64_t dM = smem_desc_sw128(sbase + OFF_M, 16, 1024);                 // K-major
        constexpr int kAtom = 8192 >> 4, kStep = 2048 >> 4, kSt = STAGE >> 4;
        constexpr uint32_t id_y = idesc_bf16_f32(128, 64, false, false);
        constexpr uint32_t id_m = idesc_bf16_f32(128, 64 * kHeads, true, false);
        int nmx = 0;
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const uint32_t st = (c % kStages) * kSt;
            if (!wait.warp(bar(bars.full[c % kStages]), c / kStages, kSsmTma)) break;
            if (!wait.warp(bar(bars.update[c & 1]), c >> 1, kSsmUpdate)) break;       // (bf16(S) is there)
            if (c >= 1 && !wait.warp(bar(bars.yread), c - 1, kSsmRead)) break;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    mma_ts(tm + TM::YI, tm + TM::SB + 8 * k, dC + st + (k >> 2) * kAtom + 2 * (k & 3), id_y, k > 0);
                mma_commit(bar(bars.cs));
            }
            __syncwarp();
            if (!wait.warp(bar(bars.mready[c & 1]), c >> 1, kSsmM)) break;
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_ss(tm + TM::YA, dX + st + k * kStep, dM + (c & 1) * kHeads * kAtom + 2 * k, id_m, k > 0);
                mma_commit(bar(bars.mx[c & 1]));
                mma_commit(bar(bars.empty[c % kStages]));
            }
            __syncwarp();
            ++nmx;
        }
        if (elect_one()) mma_commit(bar(bars.last[1]));
        __syncwarp();
        wait.drain(bar(bars.last[1]), 0, kSsmIssue);
#pragma unroll 1
        for (int c = nmx > 2 ? nmx - 2 : 0; c < nmx; ++c)
            wait.drain(bar(bars.mx[c & 1]), c >> 1, kSsmMX);
        __syncwarp();
    } else if (warp == 18) {
        // -------------------------------------------------------------- copies
        // Lanes 0..7 take a box each -- C, B, x and z, two of 64 columns -- so that the loop holds
        // one copy and one prefetch: fourteen of them in a row, fetched once a chunk, slowed
        // every other role down.
        const CUtensorMap *map = lane < 2 ? &cmap : lane < 4 ? &bmap : lane < 6 ? &xmap : &zmap;
        const int x = lane < 4 ? g * 128 + (lane & 1) * 64 : (lane & 1) ? xc1 : xc0;
        const bool staged = lane < 6 && !(LOCAL && lane < 2);
        const bool fetched = lane < (gated ? 8 : 6) && !(LOCAL && lane < 2);
        // (z two chunks behind: its place is free only when the outputs two chunks before are out, and
        // the other copies must not wait for that; at the outputs' side it is in time)
        int issued = 0, zissued = 0;
#pragma unroll 1
        for (int c = 0; c < (gated ? nch + kZBehind : nch); ++c) {
            const int t = static_cast<int>(s0) + (LOCAL ? nch - 1 - c : c) * kL;
            if (c < nch) {
                const uint32_t st = static_cast<uint32_t>(c % kStages), b = bar(bars.full[st]);
                if (c >= kStages && !wait.warp(bar(bars.empty[st]), c / kStages - 1, kSsmFree)) break;
                // (the products have read the stage; so have the outputs, for D x)
                if (!LOCAL && c >= kStages && !wait.warp(bar(bars.ydone[(c - kStages) & (kGateStages - 1)]),
                                                         (c - kStages) / kGateStages, kSsmY)) break;
                if (lane == 0) mbar_arrive_expect_tx(b, LOCAL ? STAGE - kTile : STAGE);
                __syncwarp();
                if (staged) tma_load_2d(sbase + OFF_STAGE + st * STAGE + lane * 8192, map, b, x, t);
                if (fetched && c + kPrefetch < nch) tma_prefetch_2d(map, x, LOCAL ? t - kPrefetch * kL : t + kPrefetch * kL);
                ++issued;
            }
            if (gated && c >= kZBehind) {
                // (into the staging rows that the stores two chunks before have read)
                const int k = c - kZBehind;
                if (k >= 2 && !wait.warp(bar(bars.yfree[k & 1]), (k >> 1) - 1, kSsmStage)) break;
                const uint32_t zb = bar(bars.zfull[k & 1]);
                if (lane == 0) mbar_arrive_expect_tx(zb, kTile);
                __syncwarp();
                if (lane == 6 || lane == 7)
                    tma_load_2d(sbase + OFF_Y + (k & 1) * kTile + (lane - 6) * 8192, map, zb, x, t - kZBehind * kL);
                ++zissued;
            }
        }
#pragma unroll 1
        for (int c = issued > kStages ? issued - kStages : 0; c < issued; ++c)
            wait.drain(bar(bars.full[c % kStages]), c / kStages, kSsmTma);
#pragma unroll 1
        for (int c = zissued > 2 ? zissued - 2 : 0; c < zissued; ++c)
            wait.drain(bar(bars.zfull[c & 1]), c >> 1, kSsmZ);
        __syncwarp();
    } else if (kGateWriters == 2 ? (warp == 2 || warp == 19) : warp == 2) {
        // -------------------------------------------------------------- gates
        // A lane holds tokens 2 lane and 2 lane + 1 of a chunk; one turn per chunk and head (a pair's
        // heads side by side in the local pass, where nothing else takes as long).  dt
        // is loaded two turns ahead, and its lines are brought into L2 before that: with one turn
        // between a load and its use, HBM's latency was every chunk's time.
        // (The loads are raw and unconditional: converted or masked where they are issued, each
        // waits for the one before it.)
        uint32_t d[3][2];
        const bool wide = p.dt_dtype != 1;
        auto place = [&](int c) { return LOCAL ? (c < nch ? nch - 1 - c : 0) : c; };     // of the c-th chunk
        auto fetch = [&](int i, uint32_t (&to)[2]) {
            const int t = place(i / kHeads) * kL + 2 * lane;
            const int64_t at = (s0 + (t < tokens ? t : tokens - 1)) * p.dt_stride + (PAIR && !lone ? h0 + (i & 1) : h0);
            const int64_t next = t + 1 < tokens ? at + p.dt_stride : at;
            if (wide) {
                to[0] = static_cast<const uint32_t *>(p.dt)[at];
                to[1] = static_cast<const uint32_t *>(p.dt)[next];
            } else {
                to[0] = static_cast<const uint16_t *>(p.dt)[at];
                to[1] = static_cast<const uint16_t *>(p.dt)[next];
            }
        };
        auto value = [&](uint32_t raw) { return __uint_as_float(wide ? raw : raw << 16); };
        auto ahead = [&](int c) {
            const int t = place(c) * kL + 2 * lane;
            const int64_t at = (s0 + t) * p.dt_stride + h0;
            const char *line = static_cast<const char *>(p.dt) + (p.dt_dtype == 1 ? 2 : 4) * at;
            if (t < tokens) asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
            if (t + 1 < tokens) asm volatile("prefetch.global.L2 [%0];" ::"l"(line + (p.dt_dtype == 1 ? 2 : 4) * p.dt_stride));
        };
        const int turn0 = kGateWriters == 2 && warp == 19 ? 1 : 0;
        fetch(turn0, d[0]);
        fetch(turn0 + kGateWriters, d[1]);
        float negA2[kHeads], bias[kHeads], skip[kHeads];       // (negA2: log2 decay of dt' = 1)
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
            const int h = lone ? h0 : h0 + k;
            negA2[k] = load_scalar(p.A_log, h, p.param_dtype);
            bias[k] = p.dt_bias ? load_scalar(p.dt_bias, h, p.param_dtype) : 0.0f;
            skip[k] = !LOCAL && p.D ? load_scalar(p.D, h, p.param_dtype) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kHeads; ++k) negA2[k] = max_nan(-1.4426950408889634f * ssm_rate(negA2[k]), -3.402823466e38f);
        for (int c = 1; c < kPrefetch; ++c) ahead(c);
        float later[2] = {0.0f, 0.0f};           // of the chunks behind, in the local pass
#pragma unroll 1
        for (int i = turn0; i < nch * kHeads; i += kGateWriters) {
            const int c = i / kHeads, head = PAIR ? i & 1 : 0;
            const int t0 = place(c) * kL + 2 * lane;
            fetch(i + 2 * kGateWriters, d[2]);
            if (head == 0) ahead(c + kPrefetch);
            const float b0 = PAIR && head ? bias[kHeads - 1] : bias[0];
            const float d0 = t0 < tokens ? softplus_series(value(d[0][0]) + b0) : 0.0f;
            const float d1 = t0 + 1 < tokens ? softplus_series(value(d[0][1]) + b0) : 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                d[0][k] = d[1][k];
                d[1][k] = d[2][k];
            }
            // The sums up to and including a token, and those behind it, are both summed:
            // neither is a difference of long sums.
            // (a decay below 2^-150 is zero in fp32; without the bound one such token would cost
            // the sums behind it their precision)
            const float nA = PAIR && head ? negA2[kHeads - 1] : negA2[0];
            const float a0 = max_nan(nA * d0, -160.0f), a1 = max_nan(nA * d1, -160.0f);
            float up = a0 + a1, down = up;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const float u = __shfl_up_sync(0xffffffffu, up, m), v = __shfl_down_sync(0xffffffffu, down, m);
                up += lane >= m ? u : 0.0f;
                down += lane + m < 32 ? v : 0.0f;
            }
            float before = __shfl_up_sync(0xffffffffu, up, 1), behind = __shfl_down_sync(0xffffffffu, down, 1);
            before = lane > 0 ? before : 0.0f;
            behind = lane < 31 ? behind : 0.0f;
            const float l0 = before + a0, l1 = up;
            // from a token to the end of its 8-token block
            const float n1 = __shfl_down_sync(0xffffffffu, a0 + a1, 1, 4), n2 = __shfl_down_sync(0xffffffffu, a0 + a1, 2, 4),
                        n3 = __shfl_down_sync(0xffffffffu, a0 + a1, 3, 4);
            const int q = lane & 3;
            const float rest = (q < 3 ? n1 : 0.0f) + (q < 2 ? n2 : 0.0f) + (q < 1 ? n3 : 0.0f);
            if ((kGateWriters == 2 || head == 0) && c >= kGateStages &&
                !wait.warp(bar(bars.ydone[c & (kGateStages - 1)]), c / kGateStages - 1, kSsmY)) break;
            Gates *o = gates_of(c, head);
            auto put = [&](float *to, float v0, float v1) { reinterpret_cast<float2 *>(to)[lane] = make_float2(v0, v1); };
            if (!LOCAL) {
                put(o->la, l0, l1);
                put(o->lb, l0 - __log2f(d0), l1 - __log2f(d1));
                put(o->cf, ex2(rest + a1) * d0, ex2(rest) * d1);
                put(o->e, ex2(l0), ex2(l1));
                if (lane == 0) o->D = PAIR && head ? skip[kHeads - 1] : skip[0];
            }
            const float end = LOCAL ? (head ? later[1] : later[0]) : 0.0f;
            reinterpret_cast<float2 *>(o->w[lane & 3])[lane >> 2] = make_float2(ex2(behind + a1 + end) * d0, ex2(behind + end) * d1);
            if (lane == 31) o->total = ex2(l1 + end);
            if (LOCAL) {
                const float sum = __shfl_sync(0xffffffffu, up, 31);
                later[0] += head ? 0.0f : sum;
                later[1] += head ? sum : 0.0f;
            }
            if (kGateWriters == 2 || head == kHeads - 1) warp_arrive(bar(bars.gates[c & (kGateStages - 1)]), lane);
        }
    } else if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------------- state path
        // A fragment's registers hold two neighbouring columns of rows lane / 4 and lane / 4 + 8:
        // the state goes in and out in whole 32-byte sectors.
        const int64_t frag = static_cast<int64_t>(lane_base + (lane >> 2)) * kSsmState + 2 * (lane & 3);
        float *const after = LOCAL ? args.ends + end_at * kSsmState : (last ? p.new_state + state_at : nullptr);
        const bool there = first != nullptr && !(lone && lane_base >= 64);
        bool ok = true;
        if (!LOCAL) {
#pragma unroll 1
        for (int u = 0; u < 8; ++u) {                   // 16 rows x 32 columns
            const int lh = u >> 2, q = u & 3;
            const float *from = first + frag + lh * 16 * kSsmState + 32 * q;
            uint32_t r[16];
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 v = there ? *reinterpret_cast<const float2 *>(from + k * 8 * kSsmState + 8 * m)
                                           : make_float2(0.0f, 0.0f);
                    r[4 * m + 2 * k] = __float_as_uint(v.x);
                    r[4 * m + 2 * k + 1] = __float_as_uint(v.y);
                }
            tmem_st_acc32(tmem_addr(tm, lane_base + 16 * lh, TM::S + 32 * q), r);
        }
        tmem_wait_st();
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            if (!(ok = gates_full(c))) break;
            const float decay = gates_of(c, hrow)->total;
            // Yi of the chunk before has read the copy
            if (c >= 1 && !(ok = wait.warp(bar(bars.cs), c - 1, kSsmCS))) break;
            // the state is up to date
            if (c >= 1 && !(ok = wait.warp(bar(bars.s), c - 1, kSsmS))) break;
            const uint64_t d2 = f2(decay, decay);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                uint32_t r[32], b[16];
                tmem_ld32(tmem_addr(tm, lane_base, TM::S + 32 * q), r);
                tmem_wait_ld_dep(r);
#pragma unroll
                for (int j = 0; j < 16; ++j) b[j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                tmem_st16(tmem_addr(tm, lane_base, TM::SB + 16 * q), b);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float v0, v1;
                    unf2(mul_f2(bits2(r[j], r[j + 1]), d2), v0, v1);
                    r[j] = __float_as_uint(v0);
                    r[j + 1] = __float_as_uint(v1);
                }
                tmem_st32(tmem_addr(tm, lane_base, TM::S + 32 * q), r);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(bar(bars.update[c & 1]), lane);
        }
        }
        if (LOCAL) {
            // (a thread suspended for a whole segment wakes microseconds late: along with the gates)
#pragma unroll 1
            for (int c = 0; c < nch; ++c) {
                if (!gates_full(c)) break;
                if (c + 1 < nch) warp_arrive(bar(bars.ydone[c & (kGateStages - 1)]), lane);
            }
            __syncwarp();
            // the products are all done, also after a give-up; the gates' last total is the segment's
            wait.drain(bar(bars.last[0]), 0, kSsmS);
            ok = __all_sync(0xffffffffu, wait_control()->abort == 0);
            tc_fence_after();
        } else {
            ok = ok && wait.warp(bar(bars.s), nch - 1, kSsmS);
        }
        if (LOCAL && ok) args.decays[end_at + row] = gates_of(nch - 1, hrow)->total;
        if (ok && after && !(lone && lane_base >= 64 && !LOCAL)) {
#pragma unroll 1
            for (int u = 0; u < 8; ++u) {
                const int lh = u >> 2, q = u & 3;
                float *to = after + frag + lh * 16 * kSsmState + 32 * q;
                uint32_t r[16];
                tmem_ld_frag32(tmem_addr(tm, lane_base + 16 * lh, TM::S + 32 * q), r);
                tmem_wait_ld_dep(r);
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        *reinterpret_cast<float2 *>(to + k * 8 * kSsmState + 8 * m) =
                            make_float2(__uint_as_float(r[4 * m + 2 * k]), __uint_as_float(r[4 * m + 2 * k + 1]));
            }
        }
    } else if (!LOCAL && ((warp >= 8 && warp < 12) || (warp >= 20 && warp < 24))) {
        // -------------------------------------------------------------- outputs
        // A fragment's registers hold two neighbouring tokens of one state row; stmatrix
        // writes eight rows' worth of them transposed, as 16 bytes of each token's row.
        const int mi = lane >> 3, r8 = lane & 7, i0 = warp >= 20 ? 32 : 0;      // the warp's first token
        const uint32_t yi_at = tmem_addr(tm, lane_base, TM::YI + i0), ya = TM::YA - TM::YI + (PAIR ? hrow * 64 : 0);
        const uint32_t at = (lane_base >> 6) * 8192 + sw128(i0 + 8 * (mi >> 1) + r8, ((lane_base & 63) >> 3) + (mi & 1));
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const float *e = gates_of(c, hrow)->e + i0 + 2 * (lane & 3);
            const uint32_t xs = sbase + OFF_STAGE + (c % kStages) * STAGE + ST_X;
            if (!wait.warp(bar(bars.mx[c & 1]), c >> 1, kSsmMX)) break;      // (Yi went out before Ya)
            if (p.D && !wait.warp(bar(bars.full[c % kStages]), c / kStages, kSsmTma)) break;
            uint64_t y[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {          // 16 state rows x 16 tokens
                const int lh = u & 1, hh = u >> 1;
                uint32_t yi[8], yo[8];
                tmem_ld_frag16(yi_at + (16u * lh << 16) + 16 * hh, yi);
                tmem_ld_frag16(yi_at + ya + (16u * lh << 16) + 16 * hh, yo);
                const float2 ea = *reinterpret_cast<const float2 *>(e + 16 * hh), eb = *reinterpret_cast<const float2 *>(e + 16 * hh + 8);
                tmem_wait_ld_dep(yi);
                tmem_wait_ld_dep(yo);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    y[u][k] = fma_f2(bits2(yi[2 * k], yi[2 * k + 1]), k < 2 ? f2(ea.x, ea.y) : f2(eb.x, eb.y),
                                     bits2(yo[2 * k], yo[2 * k + 1]));
            }
            // the accumulators are free for the next chunk while this one's rows are gated and stored
            tc_fence_before();
            warp_arrive(bar(bars.yread), lane);
            if (p.D) {
                const float D = gates_of(c, hrow)->D;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t xr[4];
                    ldsm_x4_t(xr, xs + ((u & 1) ? at ^ 32u : at) + (u >> 1) * 2048);
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[u][k] = fma_f2(f2(D, D), f2(bf16_lo(xr[k]), bf16_hi(xr[k])), y[u][k]);
                }
            }
            warp_arrive(bar(bars.ydone[c & (kGateStages - 1)]), lane);     // (gates and x read)
            if (gated && !wait.warp(bar(bars.zfull[c & 1]), c >> 1, kSsmZ)) break;
            // the stores two chunks before have read the staging rows (z's copy waited for them)
            if (!gated && c >= 2 && !wait.warp(bar(bars.yfree[c & 1]), (c >> 1) - 1, kSsmStage)) break;
            const uint32_t tile = sbase + OFF_Y + (c & 1) * kTile;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                // (the second 16 rows are two 16-byte words on, under the swizzle)
                const uint32_t to = tile + ((u & 1) ? at ^ 32u : at) + (u >> 1) * 2048;
                uint32_t r[4], zr[4];
                if (gated) ldsm_x4_t(zr, to);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float y0, y1;
                    unf2(y[u][k], y0, y1);
                    if (gated) {
                        y0 *= silu_approx(bf16_lo(zr[k]));
                        y1 *= silu_approx(bf16_hi(zr[k]));
                    }
                    r[k] = pack_bf16x2(y0, y1);
                }
                if (gated) __syncwarp();
                stsm_x4_t(to, r);
            }
            fence_proxy_async_smem();
            warp_arrive(bar(bars.yst[c & 1]), lane);
        }
    } else if (!LOCAL && warp == 19) {
        // -------------------------------------------------------------- output rows
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const int64_t t0 = s0 + static_cast<int64_t>(c) * kL;
            const int nt = tokens - c * kL < kL ? tokens - c * kL : kL;
            if (!wait.warp(bar(bars.yst[c & 1]), c >> 1, kSsmStage)) break;
            const uint32_t off = OFF_Y + (c & 1) * kTile;
            if (nt == kL) {
                if (lane < (lone ? 1 : 2)) {
                    tma_store_2d(&ymap, sbase + off + lane * 8192, xc0 + lane * 64, static_cast<int>(t0));
                    bulk_commit();
                    bulk_wait_read();
                }
            } else {
                // the rows behind belong to the next sequence
                const int l16 = lane & 15;
                auto *out = static_cast<__nv_bfloat16 *>(p.out) + xc0 + l16 * 8;
#pragma unroll 1
                for (int i = lane >> 4; i < nt; i += 2)
                    if (!lone || l16 < 8)
                        *reinterpret_cast<uint4 *>(out + (t0 + i) * p.heads * p.head_size) =
                            *reinterpret_cast<const uint4 *>(sm + off + (l16 >> 3) * 8192 + sw128(i, l16 & 7));
            }
            warp_arrive(bar(bars.yfree[c & 1]), lane);
        }
        if (lane < 2) bulk_wait_all();
        __syncwarp();
    } else if (!LOCAL && (warp == 16 || warp == 17 || warp == 1)) {
        // -------------------------------------------------------------- M
        // warp 16: rows and columns 0..31; 17: rows 32..63, columns 0..31; 1: rows and
        // columns 32..63.
        const int j0 = warp == 1 ? 32 : 0;
        const int block = (row - j0) >> 3;      // the 8 of its columns that hold the row's diagonal entry
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const int nt = tokens - c * kL;
            if (!gates_full(c)) break;
            // the tile has been read by Ya two chunks before
            if (c >= 2 &&
                !wait.warp(bar(bars.mx[c & 1]), (c >> 1) - 1, kSsmMX)) break;
            if (!wait.warp(bar(bars.g[c & (TM::kG - 1)]), c / TM::kG, kSsmG)) break;
            // (both heads of a pair from one read of their scores)
            float lai[kHeads], own[kHeads][8];             // the diagonal block's factors, zero above it
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const Gates *o = gates_of(c, k);
                lai[k] = o->la[row];
#pragma unroll
                for (int j = 0; j < 8; ++j) own[k][j] = j <= (row & 7) ? ex2(lai[k] - o->lb[(row & ~7) + j]) : 0.0f;
            }
            uint8_t *const tiles = sm + OFF_M + (c & 1) * kHeads * 8192;
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {                  // 8 columns
                uint32_t r[8];
                tmem_ld8(tmem_addr(tm, lane_base, TM::G + (c & (TM::kG - 1)) * 64 + j0 + 8 * q), r);
                float rf[kHeads];
#pragma unroll
                for (int k = 0; k < kHeads; ++k) rf[k] = q < block ? ex2(lai[k] - gates_of(c, k)->la[j0 + 8 * q + 7]) : 0.0f;
                tmem_wait_ld_dep(r);
                if (nt < kL) {                             // scores with rows behind the last token: zero, not x 0
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[j] = j0 + 8 * q + j < nt ? r[j] : 0u;
                }
#pragma unroll
                for (int k = 0; k < kHeads; ++k) {
                    const float4 *col = reinterpret_cast<const float4 *>(gates_of(c, k)->cf + j0 + 8 * q);
                    const float4 v0 = col[0], v1 = col[1];
                    const float f[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
                    const uint64_t rf2 = f2(rf[k], rf[k]);
                    uint32_t b[4];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        float f0, f1, m0, m1;
                        unf2(mul_f2(f2(f[j], f[j + 1]), rf2), f0, f1);
                        unf2(mul_f2(bits2(r[j], r[j + 1]), f2(q == block ? own[k][j] : f0, q == block ? own[k][j + 1] : f1)), m0, m1);
                        b[j / 2] = pack_bf16x2(m0, m1);
                    }
                    *reinterpret_cast<uint4 *>(tiles + k * 8192 + sw128(row, (j0 >> 3) + q)) = make_uint4(b[0], b[1], b[2], b[3]);
                }
            }
            tc_fence_before();
            warp_arrive(bar(bars.mread[c & (TM::kG - 1)]), lane);
            fence_proxy_async_smem();
            warp_arrive(bar(bars.mready[c & 1]), lane);
        }
    } else if ((warp >= 12 && warp < 16) || warp >= 24) {
        // -------------------------------------------------------------- w x in three terms
        // ldmatrix.trans reads the x tile [token][row] as fragments [row][token pair], the
        // layout of the TMEM operand's 32-bit columns (and stmatrix.trans writes it back).
        const int mi = lane >> 3, r8 = lane & 7, q1 = lane & 3;
        const int p0 = static_cast<int>(lane_base) + (warp >= 24 ? 16 : 0);      // the warp's first state row
        const uint32_t x0 = sbase + OFF_STAGE + ST_X + (p0 >> 6) * 8192 + sw128(8 * (mi >> 1) + r8, ((p0 & 63) >> 3) + (mi & 1));
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
            const int st = c % kStages;
            const int nt = LOCAL || tokens - c * kL > kL ? kL : tokens - c * kL;
            if (!gates_full(c)) break;
            if (!wait.warp(bar(bars.full[st]), c / kStages, kSsmTma)) break;
            if (nt < kL) {
                // Rows behind the last token, which may hold anything: zero in this warp's 16
                // columns of x and of B.
                uint8_t *bt = sm + OFF_STAGE + st * STAGE + ST_B + (p0 >> 6) * 8192;
#pragma unroll 1
                for (int i = nt * 2 + lane; i < kL * 2; i += 32) {
                    const uint32_t at = sw128(i >> 1, ((p0 & 63) >> 3) + (i & 1));
                    *reinterpret_cast<uint4 *>(bt + at) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(bt + (ST_X - ST_B) + at) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
            uint32_t w1[16], w2[16], w3[16];
            const float4 *w = reinterpret_cast<const float4 *>(gates_of(c, hrow)->w[q1]);
#pragma unroll
            for (int gp = 0; gp < 4; ++gp) {
                uint32_t x[4];
                ldsm_x4_t(x, x0 + st * STAGE + gp * 2048);
                const float4 wv = w[gp];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint64_t v = mul_f2(f2(bf16_lo(x[k]), bf16_hi(x[k])), k < 2 ? f2(wv.x, wv.y) : f2(wv.z, wv.w));
                    w1[4 * gp + k] = cut_bf2(v);
                    w2[4 * gp + k] = cut_bf2(v);
                    w3[4 * gp + k] = cut_bf2(v);
                }
            }
            if (LOCAL) warp_arrive(bar(bars.ydone[c & (kGateStages - 1)]), lane);
            // (the update of the chunk before has read the operand; all but the stores is done by then)
            if (LOCAL ? c >= 2 && !wait.warp_inline(bar(bars.g[c & 1]), (c >> 1) - 1, kSsmS)
                      : c >= 1 && !wait.warp_inline(bar(bars.s), c - 1, kSsmS)) break;
            const uint32_t w_at = tmem_addr(tm, p0, LOCAL ? TM::WL + (c & 1) * 96 : TM::W);
            tmem_st_frag32(w_at, w1);
            tmem_st_frag32(w_at + 32, w2);
            if (LOCAL) tmem_st_frag32(w_at + 64, w3);
            if (!LOCAL && !PAIR) {
#pragma unroll
                for (int gp = 0; gp < 4; ++gp)
                    stsm_x4_t(x0 - (OFF_STAGE + ST_X) + OFF_W3 + gp * 2048, *reinterpret_cast<const uint32_t(*)[4]>(w3 + 4 * gp));
                fence_proxy_async_smem();
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(bar(bars.update[c & 1]), lane);
            if (!LOCAL && PAIR) {
                // the third term in the place of bf16(S), which Yi has read
                if (!wait.warp_inline(bar(bars.cs), c, kSsmCS)) break;
                tmem_st_frag32(tmem_addr(tm, p0, TM::W3), w3);
                tmem_wait_st();
                tc_fence_before();
                warp_arrive(smem_u32(&bars.third), lane);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 32) {      // (from their sources again: no register is held for it through the roles)
        tc_fence_after();
        tmem_dealloc(tmem_slot, 512);
    }
}
// ends[slot of segment j] <- the state behind segment j, for all but a sequence's last: what
// the segment added, plus the state in front of it times the segment's decay.  One thread per
// four state elements.
constexpr int kCombineThreads = 256, kCombineCtas = kRows * kSsmState / 4 / kCombineThreads;
__global__ void __launch_bounds__(kCombineThreads) ssm_combine_kernel(const TcArgs args) {
    const int64_t chain = blockIdx.x / kCombineCtas, n = chain / args.slabs;
    const int slab = static_cast<int>(chain % args.slabs);
    const int at = static_cast<int>(blockIdx.x % kCombineCtas) * kCombineThreads + threadIdx.x;   // float4 of the block
    const int row = at / (kSsmState / 4);
    int64_t s0, s1;
    sequence_of(args.a, n, s0, s1);
    const int64_t segments = segments_of(args, s1 - s0), slot = first_slot(args, n);
    if (segments < 2) return;
    auto block = [&](int64_t j) { return (slot + j) * args.slabs + slab; };
    auto *ends = reinterpret_cast<float4 *>(args.ends);
    constexpr int kVecs = kRows * kSsmState / 4;
    const SsmArgs &p = args.a;
    const int R = p.heads / p.groups, in_group = slab % args.per_group, heads = kRows / p.head_size;
    const int h0 = slab / args.per_group * R + in_group * heads;
    float4 state = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (p.state && h0 + row / p.head_size < (slab / args.per_group + 1) * R)      // (a pair's second head may be missing)
        state = reinterpret_cast<const float4 *>(p.state + (n * p.heads + h0) * p.head_size * static_cast<int64_t>(kSsmState))[at];
    for (int64_t j = 0; j < segments - 1; ++j) {
        float4 e = ends[block(j) * kVecs + at];
        const float d = args.decays[block(j) * kRows + row];
        e.x = fmaf(d, state.x, e.x);
        e.y = fmaf(d, state.y, e.y);
        e.z = fmaf(d, state.z, e.z);
        e.w = fmaf(d, state.w, e.w);
        ends[block(j) * kVecs + at] = state = e;
    }
}

bool is_sm100() {
    int dev = 0, major = 0, minor = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    return major == 10 && minor == 0;
}

}  // namespace

// (the TMA box is 64 tokens deep; the tensors have at least as many)
bool ssm_prefill_tc_supported(int64_t total_tokens) {
    return total_tokens >= kL && total_tokens < (int64_t(1) << 31) && is_sm100();
}

namespace {

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return sms;
}

template <bool PAIR, bool LOCAL>
cudaError_t launch_pass(const CUtensorMap *maps, const TcArgs &a, int64_t slots, cudaStream_t stream) {
    const auto kernel = ssm_tc_kernel<PAIR, LOCAL>;
    const uint32_t smem = SMEM_BYTES + sizeof(WaitControl);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kernel<<<static_cast<unsigned>(slots * a.slabs), kThreads, smem, stream>>>(maps[0], maps[1], maps[2], maps[3], maps[4], a);
    return cudaGetLastError();
}

template <bool PAIR>
cudaError_t launch_passes(const CUtensorMap *maps, const TcArgs &a, int64_t slots, cudaStream_t stream) {
    if (a.ends != nullptr) {
        cudaError_t e = launch_pass<PAIR, true>(maps, a, slots, stream);
        if (e != cudaSuccess) return e;
        ssm_combine_kernel<<<static_cast<unsigned>(a.a.num_seqs * a.slabs * kCombineCtas), kCombineThreads, 0, stream>>>(a);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    return launch_pass<PAIR, false>(maps, a, slots, stream);
}

// Tokens of a segment, or 0 for no cuts, of a call with `chains` (sequence, slab) pairs, so that
// few long prompts use all SMs.  A sequence of mean length takes about 1.35 us a chunk as one;
// in k segments, at most as many as fill the SMs once, a segment's chunks take 0.75 us more
// (the local pass), and the two launches more about 14 us.  The k with the least time: 1 x
// 16,384 tokens in 32 chains 355 us uncut and 163 in four segments, 1 x 2048 in 4 chains 52
// and 29 in eight; 1 x 1024 in 32 chains stays whole at 32 us (38 in two, 31 in four).
int64_t segment_tokens(int64_t tokens, int64_t num_seqs, int64_t chains, int sms) {
    const int64_t chunks = (tokens + num_seqs * kL - 1) / (num_seqs * kL);
    const int64_t most = sms / chains < chunks / 4 ? sms / chains : chunks / 4;
    int64_t best = 0;
    double least = 1.35 * static_cast<double>(chunks);
    for (int64_t k = 2; k <= most; ++k) {
        const int64_t part = (chunks + k - 1) / k;
        const double time = (1.35 + 0.75) * static_cast<double>(part) + 14.0;
        if (time < least) {
            least = time;
            best = part * kL;
        }
    }
    return best;
}

}  // namespace

cudaError_t launch_ssm_prefill_tc(const SsmArgs &p, cudaStream_t stream) {
    const bool pair = p.head_size == 64;
    const int R = p.heads / p.groups;
    TcArgs a{p};
    a.per_group = pair ? (R + 1) / 2 : R;
    a.slabs = p.groups * a.per_group;
    a.wait_ns = wait_limit_ns();
    const int64_t chains = p.num_seqs * a.slabs;
    if (chains == 0) return cudaSuccess;
    const int sms = sm_count();
    a.segment = sms > 0 ? segment_tokens(p.rows, p.num_seqs, chains, sms) : 0;
    const bool cut = a.segment > 0 && a.segment < p.rows;
    const int64_t slots = cut ? p.rows / a.segment + p.num_seqs : p.num_seqs;
    if (slots * a.slabs > 0x7fffffffLL || chains * kCombineCtas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    CUtensorMap maps[5];
    std::memset(maps, 0, sizeof(maps));
    const int64_t wide = static_cast<int64_t>(p.heads) * p.head_size, bc = static_cast<int64_t>(p.groups) * kSsmState;
    if (!make_tmap_rows_bf16(&maps[0], p.x, p.rows, wide, p.x_stride) ||
        !make_tmap_rows_bf16(&maps[1], p.B, p.rows, bc, p.B_stride) ||
        !make_tmap_rows_bf16(&maps[2], p.C, p.rows, bc, p.C_stride) ||
        (p.z && !make_tmap_rows_bf16(&maps[3], p.z, p.rows, wide, p.z_stride)) ||
        !make_tmap_rows_bf16(&maps[4], p.out, p.rows, wide, wide))
        return cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess, ef = cudaSuccess;
    if (cut) {
        void *ws = nullptr;
        const size_t blocks = static_cast<size_t>(slots) * a.slabs;
        if ((e = pool_alloc(&ws, blocks * (kRows * kSsmState + kRows) * sizeof(float), stream)) != cudaSuccess) return e;
        a.ends = static_cast<float *>(ws);
        a.decays = a.ends + blocks * kRows * kSsmState;
    }
    e = pair ? launch_passes<true>(maps, a, slots, stream) : launch_passes<false>(maps, a, slots, stream);
    if (cut) ef = cudaFreeAsync(a.ends, stream);
    return e != cudaSuccess ? e : ef;
}

}  // namespace gdn
