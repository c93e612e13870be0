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
//   Ya^T = x^T bf16(M)^T         the chunk's own part; D sits on M's diagonal
//   S   += (w x)^T B             w x split into bf16 hi + lo (two products), so the fp32
//                                state loses 2^-17 per term, not 2^-9
// M's exponentials: la_i - la_j <= 0 on and below the diagonal, so none overflows; the block
// of rows 32..63 and columns 0..31 factors into exp(la_i - la_31) exp(la_31 - la_j), both at
// most 1, and only the two diagonal 32 x 32 blocks take one exponential per element.
//
// Roles (20 warps), handing chunks to each other through mbarriers:
//   warp 0       allocates TMEM; lane 0 issues every MMA as soon as its inputs are ready,
//                the state update first
//   warp 1       copies (TMA), two stages of C, B and x, and of z
//   warps 2, 3   the chunk's gates, one head each
//   warps 4-7    state path: S -> bf16 copy (TMEM operand of Yi) and the decay of S
//   warps 8-11   outputs: Yi, Ya from TMEM, the gate z, bf16 rows through shared memory
//   warps 12, 13, 17   M, a 32 x 32 block each
//   warps 14, 15, 18, 19   w x hi / lo; the rows behind the last token set to zero
//
// Every wait is bounded as in gdn_prefill_tc.cu: one that gives up records its site in the
// device status word and raises a shared flag, every role stops at its next wait, the
// issuing threads wait (bounded) for their own MMAs and copies, and the CTA frees TMEM.
#include <cuda_bf16.h>
#include <cstring>

#include "gdn_ssm_common.cuh"
#include "sm100.cuh"
#include "tma_host.h"

namespace gdn {

namespace {

using namespace sm100;

constexpr int kL = 64;              // tokens of a chunk
constexpr int kThreads = 640;
constexpr int kRows = 128;          // state rows of a CTA
constexpr int kSplitWarps = 4, kMWarps = 3;

// Shared memory (bytes from the 1024-aligned base).  Tiles are 64 rows of 64 bf16 (one
// 128-byte swizzled atom, 8 KB), two atoms side by side.
constexpr uint32_t kTile = 16 * 1024;
constexpr uint32_t OFF_STAGE = 0;                       // 2 x [C | B | x]
constexpr uint32_t STAGE = 3 * kTile;
constexpr uint32_t ST_C = 0, ST_B = kTile, ST_X = 2 * kTile;
constexpr uint32_t OFF_WX = OFF_STAGE + 2 * STAGE;      // [hi | lo], each as x
constexpr uint32_t OFF_M = OFF_WX + 2 * kTile;          // [head][i][j], K-major, 8 KB each
constexpr uint32_t OFF_Y = OFF_M + kTile;               // bf16 [64][128] output rows
constexpr uint32_t OFF_GATE = OFF_Y + kTile;            // 2 x 2 heads x Gates
constexpr uint32_t GATE = 1536;
constexpr uint32_t OFF_Z = OFF_GATE + 6 * 1024;         // 2 x z, only with the output gate
constexpr uint32_t SMEM_PLAIN = OFF_Z, SMEM_GATED = OFF_Z + 2 * kTile;
static_assert(OFF_Z % 1024 == 0 && SMEM_GATED <= 227 * 1024, "shared memory map");

struct Gates {
    float la[64];    // sum of the log2 decays from the start of the token's 32-token half
    float dt[64];    // dt'
    float e[64];     // exp(la_i) from the start of the chunk
    float w[64];     // exp(la_63 - la_j) dt'_j
    float cf[32];    // exp(la_31 - la_j) dt'_j, j < 32
    float rf[32];    // exp(la_{32 + i} - la_31)
    float total;     // exp(la_63)
};
static_assert(sizeof(Gates) <= GATE, "gate block");

// TMEM columns (all 512 allocated).
constexpr uint32_t TM_S = 0;       // [0, 128)   fp32 state
constexpr uint32_t TM_SB = 128;    // 2 x 64     bf16x2 copy of the state in front of a chunk
constexpr uint32_t TM_G = 256;     // [256, 320) G, lanes 0..63
constexpr uint32_t TM_YI = 320;    // [320, 384) Yi^T
constexpr uint32_t TM_YA = 384;    // [384, 512) Ya^T: 64 columns, or 64 per head of a pair

enum WaitSite { kSsmTma = 41, kSsmZ = 42, kSsmGates = 43, kSsmG = 44, kSsmM = 45, kSsmS = 46, kSsmCS = 47,
                kSsmMX = 48, kSsmIssue = 49, kSsmY = 50, kSsmStage = 51, kSsmFree = 52 };
constexpr uint64_t kDrainNs = 2000000000ull;
constexpr uint32_t kMaxSuspendNs = 1000000;

struct TcArgs {
    SsmArgs a;
    int slabs, per_group;    // CTAs per sequence, per group
    uint64_t wait_ns;
};

struct Bars {
    uint64_t full[2], empty[2], zfull[2], gates[2], ydone[2], cs[2];
    uint64_t g, mread, mready, mx, s, sready, split, yread, yst, yfree;
};

struct Waiter {
    volatile int *abort;
    int *status;
    uint64_t limit;

    __device__ __forceinline__ bool one(uint32_t bar, uint32_t parity, int site) const {
        if (mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = global_timer_ns();
        const uint32_t hint = limit < kMaxSuspendNs ? static_cast<uint32_t>(limit) : kMaxSuspendNs;
        for (;;) {
            if (mbar_try_wait_hint(bar, parity, hint)) return true;
            if (*abort) return false;
            if (global_timer_ns() - t0 > limit) {
                give_up(site);
                return false;
            }
        }
    }
    __device__ __forceinline__ void give_up(int site) const {
        if (status) atomicCAS(status, 0, site);
        *abort = 1;
    }
    // The whole warp; reconverges it for the next .aligned tcgen05 instruction.
    __device__ __forceinline__ bool warp(uint32_t bar, uint32_t parity, int site) const {
        const bool ok = one(bar, parity, site);
        __syncwarp();
        tc_fence_after();
        return __all_sync(0xffffffffu, ok);
    }
    // This CTA's own copies and MMAs, also after a give-up.
    __device__ __forceinline__ void drain(uint32_t bar, uint32_t parity, int site) const {
        volatile int never = 0;
        Waiter w{&never, status, kDrainNs};
        w.one(bar, parity, site);
    }
};

__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// PAIR: two heads of 64 rows; else one head of 128.
template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
ssm_tc_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap bmap,
              const __grid_constant__ CUtensorMap cmap, const __grid_constant__ CUtensorMap zmap, const TcArgs args) {
    extern __shared__ __align__(1024) uint8_t sm[];
    __shared__ Bars bars;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const SsmArgs &p = args.a;
    constexpr int kHeads = PAIR ? 2 : 1;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t lane_base = static_cast<uint32_t>(warp & 3) * 32;
    const int row = static_cast<int>(lane_base) + lane;    // this thread's TMEM lane
    const int64_t n = blockIdx.x / args.slabs;
    const int slab = static_cast<int>(blockIdx.x % args.slabs);
    const int g = slab / args.per_group, R = p.heads / p.groups;
    const int h0 = g * R + (slab % args.per_group) * kHeads;
    const bool lone = PAIR && (slab % args.per_group) * 2 + 1 >= R;   // a pair's second head is missing
    const int64_t T = p.rows;
    if (tid == 0 && slab == 0) check_seq_bounds(p.cu_seqlens, n, p.num_seqs, T, p.status);
    int64_t s0 = p.cu_seqlens[n], s1 = p.cu_seqlens[n + 1];
    s0 = s0 < 0 ? 0 : (s0 > T ? T : s0);
    s1 = s1 < s0 ? s0 : (s1 > T ? T : s1);
    const int nch = static_cast<int>((s1 - s0 + kL - 1) / kL);
    const bool gated = p.z != nullptr;
    const uint32_t sbase = smem_u32(sm);
    auto bar = [&](const uint64_t &b) { return smem_u32(&b); };
    const Waiter wait{&abort_flag, p.status, args.wait_ns};

    // this thread's state row: of head h0, or for the second half of a pair of head h0 + 1
    const int hrow = PAIR ? row >> 6 : 0;
    const bool dead = lone && hrow == 1;
    const int64_t state_at =
        ((n * p.heads + h0 + hrow) * p.head_size + (PAIR ? row & 63 : row)) * static_cast<int64_t>(kSsmState);

    if (nch == 0) {
        // An empty sequence keeps its state (or starts at zero).
        const int64_t base = (n * p.heads + h0) * p.head_size * static_cast<int64_t>(kSsmState);
        const int vecs = (lone ? 64 : kRows) * kSsmState / 4;
        for (int i = tid; i < vecs; i += kThreads)
            reinterpret_cast<float4 *>(p.new_state + base)[i] =
                p.state ? reinterpret_cast<const float4 *>(p.state + base)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        return;
    }
    if (warp == 0) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                mbar_init(bar(bars.full[i]), 1);
                mbar_init(bar(bars.empty[i]), 1);
                mbar_init(bar(bars.zfull[i]), 1);
                mbar_init(bar(bars.gates[i]), kHeads);
                mbar_init(bar(bars.ydone[i]), 4);
                mbar_init(bar(bars.cs[i]), 1);
            }
            mbar_init(bar(bars.g), 1);
            mbar_init(bar(bars.mread), kMWarps);
            mbar_init(bar(bars.mready), kMWarps);
            mbar_init(bar(bars.mx), 1);
            mbar_init(bar(bars.s), 1);
            mbar_init(bar(bars.sready), 4);
            mbar_init(bar(bars.split), kSplitWarps);
            mbar_init(bar(bars.yread), 4);
            mbar_init(bar(bars.yst), 4);
            mbar_init(bar(bars.yfree), 4);
            abort_flag = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(smem_u32(&tmem_slot), 512);
        tmem_relinquish();
    }
    // M's upper right blocks stay zero
    for (int i = tid; i < static_cast<int>(kTile / 16); i += kThreads)
        reinterpret_cast<uint4 *>(sm + OFF_M)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_slot;
    auto gates_of = [&](int c, int head) -> Gates * {
        return reinterpret_cast<Gates *>(sm + OFF_GATE + ((c & 1) * 2 + head) * GATE);
    };

    if (warp == 0) {
        // -------------------------------------------------------------- MMA issue
        if (lane == 0) {
            const uint64_t dC = smem_desc_sw128(sbase + OFF_STAGE + ST_C, 16, 1024);      // K-major
            const uint64_t dBk = smem_desc_sw128(sbase + OFF_STAGE + ST_B, 16, 1024);     // K-major
            const uint64_t dBm = smem_desc_sw128(sbase + OFF_STAGE + ST_B, 8192, 1024);   // MN-major
            const uint64_t dX = smem_desc_sw128(sbase + OFF_STAGE + ST_X, 8192, 1024);    // MN-major
            const uint64_t dW = smem_desc_sw128(sbase + OFF_WX, 8192, 1024);              // MN-major
            const uint64_t dM = smem_desc_sw128(sbase + OFF_M, 16, 1024);                 // K-major
            constexpr uint32_t kAtom = 8192 >> 4, kStep = 2048 >> 4, kSt = STAGE >> 4, kLo = kTile >> 4;
            constexpr uint32_t id_g = idesc_bf16_f32(128, 64, false, false);
            constexpr uint32_t id_s = idesc_bf16_f32(128, 128, true, true);
            constexpr uint32_t id_m = idesc_bf16_f32(128, 64 * kHeads, true, false);
            int ng = 0, nmx = 0, ncs = 0, ns = 0, nfree = 0;
            bool ok = true;
            uint32_t idle = 0;
            uint64_t t_idle = 0;
            while (ok && nfree < nch) {
                bool progress = false;
                // A barrier is looked at by the parity of its phase, so only while it cannot be
                // two phases on: where the state update of a chunk is out (ns ahead), its
                // inputs' barriers were seen then and may have moved on since.
                // The state update (its stage has landed when G of the chunk is out):
                if (ns < ng && mbar_test_wait(bar(bars.sready), ns & 1) && mbar_test_wait(bar(bars.split), ns & 1)) {
                    tc_fence_after();
                    const uint32_t st = (ns & 1) * kSt;
#pragma unroll
                    for (int part = 0; part < 2; ++part)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ss(tm + TM_S, dW + part * kLo + k * kStep, dBm + st + k * kStep, id_s, 1);
                    mma_commit(bar(bars.s));
                    ++ns;
                    progress = true;
                }
                if (ncs < ng && (ncs < ns || mbar_test_wait(bar(bars.sready), ncs & 1)) &&
                    (ncs == 0 || mbar_test_wait(bar(bars.yread), (ncs - 1) & 1))) {
                    tc_fence_after();
                    const uint32_t st = (ncs & 1) * kSt;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_ts(tm + TM_YI, tm + TM_SB + (ncs & 1) * 64 + 8 * k, dC + st + (k >> 2) * kAtom + 2 * (k & 3),
                               id_g, k > 0);
                    mma_commit(bar(bars.cs[ncs & 1]));
                    ++ncs;
                    progress = true;
                }
                if (nmx < ng && mbar_test_wait(bar(bars.mready), nmx & 1) &&
                    (nmx < ns || mbar_test_wait(bar(bars.split), nmx & 1)) &&
                    (nmx == 0 || mbar_test_wait(bar(bars.yread), (nmx - 1) & 1))) {
                    tc_fence_after();
                    const uint32_t st = (nmx & 1) * kSt;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss(tm + TM_YA, dX + st + k * kStep, dM + 2 * k, id_m, k > 0);
                    mma_commit(bar(bars.mx));
                    ++nmx;
                    progress = true;
                }
                // G goes at most one chunk ahead of the slowest other product (the barriers
                // of a chunk are looked at by parity)
                if (ng < nch && ng <= nfree + 1 && mbar_test_wait(bar(bars.full[ng & 1]), (ng >> 1) & 1) &&
                    (ng == 0 || mbar_test_wait(bar(bars.mread), (ng - 1) & 1))) {
                    tc_fence_after();
                    const uint32_t st = (ng & 1) * kSt;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        mma_ss(tm + TM_G, dC + st + (k >> 2) * kAtom + 2 * (k & 3), dBk + st + (k >> 2) * kAtom + 2 * (k & 3),
                               id_g, k > 0);
                    mma_commit(bar(bars.g));
                    ++ng;
                    progress = true;
                }
                if (nfree < ns && nfree < ncs && nfree < nmx) {
                    mma_commit(bar(bars.empty[nfree & 1]));
                    ++nfree;
                }
                if (progress) {
                    idle = 0;
                } else if ((++idle & 255u) == 0) {
                    if (idle == 256) {
                        t_idle = global_timer_ns();
                    } else if (*wait.abort) {
                        ok = false;
                    } else if (global_timer_ns() - t_idle > wait.limit) {
                        wait.give_up(kSsmIssue);
                        ok = false;
                    }
                }
            }
            // No MMA or barrier arrive is in flight when the CTA leaves.
            if (ng) wait.drain(bar(bars.g), (ng - 1) & 1, kSsmG);
            for (int c = ncs > 2 ? ncs - 2 : 0; c < ncs; ++c) wait.drain(bar(bars.cs[c & 1]), (c >> 1) & 1, kSsmCS);
            if (nmx) wait.drain(bar(bars.mx), (nmx - 1) & 1, kSsmMX);
            if (ns) wait.drain(bar(bars.s), (ns - 1) & 1, kSsmS);
            for (int c = nfree > 2 ? nfree - 2 : 0; c < nfree; ++c)
                wait.drain(bar(bars.empty[c & 1]), (c >> 1) & 1, kSsmFree);
        }
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------------------- copies
        if (lane == 0) {
            const int xc0 = PAIR ? h0 * 64 : h0 * 128;
            const int xc1 = lone ? xc0 : xc0 + 64;      // (a lone head twice: its copy is not stored)
            int issued = 0, zissued = 0;
            for (int c = 0; c < nch; ++c) {
                const int st = c & 1, t = static_cast<int>(s0 + static_cast<int64_t>(c) * kL);
                if (c >= 2 && !wait.one(bar(bars.empty[st]), ((c - 2) >> 1) & 1, kSsmFree)) break;
                const uint32_t base = sbase + OFF_STAGE + st * STAGE, b = bar(bars.full[st]);
                mbar_arrive_expect_tx(b, STAGE);
                tma_load_2d(base + ST_C, &cmap, b, g * 128, t);
                tma_load_2d(base + ST_C + 8192, &cmap, b, g * 128 + 64, t);
                tma_load_2d(base + ST_B, &bmap, b, g * 128, t);
                tma_load_2d(base + ST_B + 8192, &bmap, b, g * 128 + 64, t);
                tma_load_2d(base + ST_X, &xmap, b, xc0, t);
                tma_load_2d(base + ST_X + 8192, &xmap, b, xc1, t);
                ++issued;
                if (gated) {
                    if (c >= 2 && !wait.one(bar(bars.ydone[st]), ((c - 2) >> 1) & 1, kSsmY)) break;
                    const uint32_t zb = bar(bars.zfull[st]);
                    mbar_arrive_expect_tx(zb, kTile);
                    tma_load_2d(sbase + OFF_Z + st * kTile, &zmap, zb, xc0, t);
                    tma_load_2d(sbase + OFF_Z + st * kTile + 8192, &zmap, zb, xc1, t);
                    ++zissued;
                }
            }
            for (int c = issued > 2 ? issued - 2 : 0; c < issued; ++c)
                wait.drain(bar(bars.full[c & 1]), (c >> 1) & 1, kSsmTma);
            for (int c = zissued > 2 ? zissued - 2 : 0; c < zissued; ++c)
                wait.drain(bar(bars.zfull[c & 1]), (c >> 1) & 1, kSsmZ);
        }
        __syncwarp();
    } else if (warp < 2 + kHeads) {
        // -------------------------------------------------------------- gates of one head
        const int head = warp - 2;
        const int h = lone ? h0 : h0 + head;
        const float negA2 = -expf(load_scalar(p.A_log, h, p.param_dtype)) * 1.4426950408889634f;   // log2 decays
        auto step_of = [&](int64_t t) { return t < s1 ? ssm_step(p, t, h) : 0.0f; };
        float d0 = step_of(s0 + lane), d1 = step_of(s0 + 32 + lane);
        for (int c = 0; c < nch; ++c) {
            const float a0 = negA2 * d0, a1 = negA2 * d1;
            // sums up to and including a token, and behind it, of each 32-token half: both
            // directions are summed, none is a difference of long sums
            float p0 = a0, p1 = a1, q0 = a0, q1 = a1;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const float u0 = __shfl_up_sync(0xffffffffu, p0, m), u1 = __shfl_up_sync(0xffffffffu, p1, m);
                const float v0 = __shfl_down_sync(0xffffffffu, q0, m), v1 = __shfl_down_sync(0xffffffffu, q1, m);
                if (lane >= m) {
                    p0 += u0;
                    p1 += u1;
                }
                if (lane + m < 32) {
                    q0 += v0;
                    q1 += v1;
                }
            }
            const float t0 = __shfl_sync(0xffffffffu, p0, 31), t1 = __shfl_sync(0xffffffffu, p1, 31);
            q0 = __shfl_down_sync(0xffffffffu, q0, 1);
            q1 = __shfl_down_sync(0xffffffffu, q1, 1);
            if (lane == 31) q0 = q1 = 0.0f;
            if (c >= 2 && !wait.warp(bar(bars.ydone[c & 1]), ((c - 2) >> 1) & 1, kSsmY)) break;
            Gates *o = gates_of(c, head);
            o->la[lane] = p0;
            o->la[lane + 32] = p1;
            o->dt[lane] = d0;
            o->dt[lane + 32] = d1;
            o->e[lane] = exp2f(p0);
            o->e[lane + 32] = exp2f(t0 + p1);
            o->w[lane] = exp2f(q0 + t1) * d0;
            o->w[lane + 32] = exp2f(q1) * d1;
            o->cf[lane] = exp2f(q0) * d0;
            o->rf[lane] = exp2f(p1);
            if (lane == 0) o->total = exp2f(t0 + t1);
            warp_arrive(bar(bars.gates[c & 1]), lane);
            if (c + 1 < nch) {
                const int64_t t = s0 + static_cast<int64_t>(c + 1) * kL + lane;
                d0 = step_of(t);
                d1 = step_of(t + 32);
            }
        }
    } else if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------------- state path
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
            uint32_t r[32];
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const float4 x = p.state && !dead ? *reinterpret_cast<const float4 *>(p.state + state_at + 32 * q + j)
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
                r[j] = __float_as_uint(x.x); r[j + 1] = __float_as_uint(x.y);
                r[j + 2] = __float_as_uint(x.z); r[j + 3] = __float_as_uint(x.w);
            }
            tmem_st32(tmem_addr(tm, lane_base, TM_S + 32 * q), r);
        }
        tmem_wait_st();
        bool ok = true;
        for (int c = 0; c < nch; ++c) {
            if (!(ok = wait.warp(bar(bars.gates[c & 1]), (c >> 1) & 1, kSsmGates))) break;
            const float decay = gates_of(c, hrow)->total;
            if (c >= 2 && !(ok = wait.warp(bar(bars.cs[c & 1]), ((c - 2) >> 1) & 1, kSsmCS))) break;
            if (c >= 1 && !(ok = wait.warp(bar(bars.s), (c - 1) & 1, kSsmS))) break;
            const uint64_t d2 = f2(decay, decay);
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                uint32_t r[32], b[16];
                tmem_ld32(tmem_addr(tm, lane_base, TM_S + 32 * q), r);
                tmem_wait_ld_dep(r);
#pragma unroll
                for (int j = 0; j < 16; ++j) b[j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                tmem_st16(tmem_addr(tm, lane_base, TM_SB + (c & 1) * 64 + 16 * q), b);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    float v0, v1;
                    unf2(mul_f2(f2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), d2), v0, v1);
                    r[j] = __float_as_uint(v0);
                    r[j + 1] = __float_as_uint(v1);
                }
                tmem_st32(tmem_addr(tm, lane_base, TM_S + 32 * q), r);
            }
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(bar(bars.sready), lane);
        }
        if (ok && wait.warp(bar(bars.s), (nch - 1) & 1, kSsmS)) {
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                uint32_t r[32];
                tmem_ld32(tmem_addr(tm, lane_base, TM_S + 32 * q), r);
                tmem_wait_ld_dep(r);
                if (!dead) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        *reinterpret_cast<float4 *>(p.new_state + state_at + 32 * q + j) =
                            make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                                        __uint_as_float(r[j + 3]));
                }
                __syncwarp();
            }
        }
    } else if (warp >= 8 && warp < 12) {
        // -------------------------------------------------------------- outputs
        const int yw = warp - 8, l16 = lane & 15, half = lane >> 4;
        const uint32_t ya = TM_YA + (PAIR ? hrow * 64 : 0);
        uint16_t *so = reinterpret_cast<uint16_t *>(sm + OFF_Y);
        auto *out = static_cast<__nv_bfloat16 *>(p.out) + static_cast<int64_t>(h0) * p.head_size + l16 * 8;
        const bool stores = !lone || l16 < 8;
        for (int c = 0; c < nch; ++c) {
            const int st = c & 1;
            const int64_t t0 = s0 + static_cast<int64_t>(c) * kL;
            const int nt = static_cast<int>(s1 - t0 < kL ? s1 - t0 : kL);
            const float *e = gates_of(c, hrow)->e;
            if (gated && !wait.warp(bar(bars.zfull[st]), (c >> 1) & 1, kSsmZ)) break;
            if (!wait.warp(bar(bars.cs[c & 1]), (c >> 1) & 1, kSsmCS)) break;
            if (!wait.warp(bar(bars.mx), c & 1, kSsmMX)) break;
            // the stores of the chunk before have read the staging rows
            if (c > 0 && !wait.warp(bar(bars.yfree), (c - 1) & 1, kSsmStage)) break;
            const uint8_t *zt = sm + OFF_Z + st * kTile + (row >> 6) * 8192 + (row & 7) * 2;
            const int zc = (row & 63) >> 3;
#pragma unroll 1
            for (int hf = 0; hf < 2; ++hf) {
                uint32_t yi[32], yo[32];
                tmem_ld32(tmem_addr(tm, lane_base, TM_YI + 32 * hf), yi);
                tmem_ld32(tmem_addr(tm, lane_base, ya + 32 * hf), yo);
                tmem_wait_ld_dep(yi);
                tmem_wait_ld_dep(yo);
                if (hf == 1) {
                    tc_fence_before();
                    warp_arrive(bar(bars.yread), lane);
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const int i = 32 * hf + j;
                    float y0, y1;
                    unf2(fma_f2(f2(__uint_as_float(yi[j]), __uint_as_float(yi[j + 1])), f2(e[i], e[i + 1]),
                                f2(__uint_as_float(yo[j]), __uint_as_float(yo[j + 1]))), y0, y1);
                    if (gated) {
                        y0 *= ssm_silu(__bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(zt + sw128(i, zc))));
                        y1 *= ssm_silu(__bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(zt + sw128(i + 1, zc))));
                    }
                    const uint32_t pk = pack_bf16x2(y0, y1);
                    so[i * kRows + row] = static_cast<uint16_t>(pk);
                    so[(i + 1) * kRows + row] = static_cast<uint16_t>(pk >> 16);
                }
            }
            warp_arrive(bar(bars.ydone[st]), lane);     // (gates and z read)
            warp_arrive(bar(bars.yst), lane);
            if (!wait.warp(bar(bars.yst), c & 1, kSsmStage)) break;
#pragma unroll 2
            for (int u = 0; u < 8; ++u) {
                const int i = 16 * yw + 2 * u + half;
                const uint4 v = *reinterpret_cast<const uint4 *>(so + i * kRows + l16 * 8);
                if (i < nt && stores)
                    *reinterpret_cast<uint4 *>(out + (t0 + i) * p.heads * p.head_size) = v;
            }
            warp_arrive(bar(bars.yfree), lane);
        }
    } else if (warp == 12 || warp == 13 || warp == 17) {
        // -------------------------------------------------------------- M
        // warp 12: rows and columns 0..31; 13: rows 32..63, columns 0..31; 17: rows and
        // columns 32..63.
        const bool diag = warp != 13;
        const int i = row, j0 = warp == 17 ? 32 : 0;
        float D[kHeads];
#pragma unroll
        for (int k = 0; k < kHeads; ++k) D[k] = p.D ? load_scalar(p.D, lone ? h0 : h0 + k, p.param_dtype) : 0.0f;
        for (int c = 0; c < nch; ++c) {
            if (!wait.warp(bar(bars.gates[c & 1]), (c >> 1) & 1, kSsmGates)) break;
            if (!wait.warp(bar(bars.g), c & 1, kSsmG)) break;
            uint32_t r[32];
            tmem_ld32(tmem_addr(tm, lane_base, TM_G + j0), r);
            tmem_wait_ld_dep(r);
            tc_fence_before();
            warp_arrive(bar(bars.mread), lane);
            if (c >= 1 && !wait.warp(bar(bars.mx), (c - 1) & 1, kSsmMX)) break;
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const Gates *o = gates_of(c, k);
                const float lai = o->la[i], rfi = o->rf[lane];
                uint8_t *dst = sm + OFF_M + k * 8192;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t b[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = 8 * q + 2 * e;
                        float v[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float gv = __uint_as_float(r[j + u]);
                            if (diag) {
                                const float m = gv * (exp2f(lai - o->la[j0 + j + u]) * o->dt[j0 + j + u]);
                                v[u] = j + u < lane ? m : (j + u == lane ? m + D[k] : 0.0f);
                            } else {
                                v[u] = gv * (rfi * o->cf[j + u]);
                            }
                        }
                        b[e] = pack_bf16x2(v[0], v[1]);
                    }
                    *reinterpret_cast<uint4 *>(dst + sw128(i, (j0 >> 3) + q)) = make_uint4(b[0], b[1], b[2], b[3]);
                }
            }
            fence_proxy_async_smem();
            warp_arrive(bar(bars.mready), lane);
        }
    } else if (warp == 14 || warp == 15 || warp == 18 || warp == 19) {
        // -------------------------------------------------------------- w x, hi and lo
        const int t = (warp < 16 ? warp - 14 : warp - 16) * 32 + lane;     // 0..127
        for (int c = 0; c < nch; ++c) {
            const int st = c & 1;
            const int64_t t0 = s0 + static_cast<int64_t>(c) * kL;
            const int nt = static_cast<int>(s1 - t0 < kL ? s1 - t0 : kL);
            if (!wait.warp(bar(bars.gates[st]), (c >> 1) & 1, kSsmGates)) break;
            if (!wait.warp(bar(bars.full[st]), (c >> 1) & 1, kSsmTma)) break;
            if (c >= 1 && !wait.warp(bar(bars.s), (c - 1) & 1, kSsmS)) break;
            uint8_t *xs = sm + OFF_STAGE + st * STAGE + ST_X, *bs = sm + OFF_STAGE + st * STAGE + ST_B;
#pragma unroll 2
            for (int u = 0; u < 8; ++u) {
                const int at = u * 128 + t, j = (at >> 3) & 63;     // 16-byte word; atom at >> 9, token j
                const float w = gates_of(c, PAIR ? at >> 9 : 0)->w[j];
                uint32_t hi[4] = {}, lo[4] = {};
                if (j < nt) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(xs + at * 16);
                    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
                    const uint64_t w2 = f2(w, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v0, v1;
                        unf2(mul_f2(f2(bf16_lo(x[e]), bf16_hi(x[e])), w2), v0, v1);
                        split2_bf16_f2(v0, v1, hi[e], lo[e]);
                    }
                } else {
                    // rows behind the last token: other sequences' or none
                    *reinterpret_cast<uint4 *>(xs + at * 16) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(bs + at * 16) = make_uint4(0, 0, 0, 0);
                }
                *reinterpret_cast<uint4 *>(sm + OFF_WX + at * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(sm + OFF_WX + kTile + at * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_proxy_async_smem();
            warp_arrive(bar(bars.split), lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tm, 512);
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

cudaError_t launch_ssm_prefill_tc(const SsmArgs &p, cudaStream_t stream) {
    const bool pair = p.head_size == 64;
    const int R = p.heads / p.groups;
    TcArgs a{p};
    a.per_group = pair ? (R + 1) / 2 : R;
    a.slabs = p.groups * a.per_group;
    a.wait_ns = wait_limit_ns();
    const int64_t ctas = p.num_seqs * a.slabs;
    if (ctas == 0) return cudaSuccess;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    CUtensorMap maps[4];
    std::memset(maps, 0, sizeof(maps));
    const int64_t wide = static_cast<int64_t>(p.heads) * p.head_size, bc = static_cast<int64_t>(p.groups) * kSsmState;
    if (!make_tmap_rows_bf16(&maps[0], p.x, p.rows, wide, p.x_stride) ||
        !make_tmap_rows_bf16(&maps[1], p.B, p.rows, bc, p.B_stride) ||
        !make_tmap_rows_bf16(&maps[2], p.C, p.rows, bc, p.C_stride) ||
        (p.z && !make_tmap_rows_bf16(&maps[3], p.z, p.rows, wide, p.z_stride)))
        return cudaErrorInvalidValue;
    const auto kernel = pair ? ssm_tc_kernel<true> : ssm_tc_kernel<false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_GATED);
    if (e != cudaSuccess) return e;
    kernel<<<static_cast<unsigned>(ctas), kThreads, p.z ? SMEM_GATED : SMEM_PLAIN, stream>>>(maps[0], maps[1], maps[2],
                                                                                             maps[3], a);
    return cudaGetLastError();
}

}  // namespace gdn
