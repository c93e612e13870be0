// gdn_conv.cu -- the short depthwise causal convolution in front of a linear-attention
// layer's recurrence (not part of the reference, which starts at q, k and v):
//
//   y[t][c] = act(bias[c] + sum_{w < W} weight[c][w] * x[t - (W-1) + w][c]),   W = 2, 3, 4,
//
// per packed sequence, where the W-1 rows in front of its first token are its state (zero
// without one), act is the identity or silu(y) = y / (1 + exp(-y)), and the new state is
// the last W-1 rows of [state; x].  fp32 arithmetic from bf16 rows, one rounding of y.
//
// Both kernels are HBM-bound (4 bytes a token and channel against 2 W flops and one silu, of
// whose two hardware functions an SM does 16 a cycle: 0.24 of the 0.33 ms that 65,536 x 8192
// take to read and write).  A thread owns 4 channels (8 bytes of a row) and a run of
// consecutive tokens, so the window slides through its registers: every row is read from HBM
// once, plus W-1 rows of overlap per run that mostly hit in L2.  Four channels and not eight,
// whose weights and window alone took 96 registers: with 12 warps an SM the loads in flight
// covered half of HBM's latency (0.68 ms).  The rows ahead wait in a ring in shared memory
// that every thread fills (cp.async) and reads for itself, without a barrier: loaded into
// registers a batch at a time, the loads of a batch did not overlap the arithmetic of the one
// before (0.456 ms).  65,536 x 8192: 0.337 ms, 6.4 TB/s; batches of 8 rows or a ring of 24 cost
// resident blocks (0.40 to 0.42 ms), batches of 2 take 0.37 ms.  A few short prompts (1280
// tokens) take 12 us, most of it the latency of three dependent reads (offsets, rows, window).
//
// Decode (512 x 8192, width 4, with a bias): 13 us, 5.2 TB/s, a thread's runs short enough to
// fill the SMs, since its weights are read once a run; 4 x 8192: 2.5 us, a launch's latency.
#include "gdn_common.cuh"
#include "gdn_launch.h"
#include "gdn_mma_sync.cuh"

namespace gdn {

namespace {

constexpr int kVec = 4;            // channels of a thread
constexpr int kConvThreads = 128;
constexpr int kBatchRows = 4;      // rows a thread copies at once
constexpr int kBatches = 4;        // batches of the ring: one in use, the others on their way

struct Row {                       // 4 channels as packed fp32 pairs
    uint64_t v[2];
};

__device__ __forceinline__ Row unpack_row(uint2 w) {
    Row r;
    r.v[0] = f2(bf16_lo(w.x), bf16_hi(w.x));
    r.v[1] = f2(bf16_lo(w.y), bf16_hi(w.y));
    return r;
}

// 8 bytes global -> shared, asynchronously.
__device__ __forceinline__ void copy_row(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint2 load_row(const __nv_bfloat16 *p) { return __ldg(reinterpret_cast<const uint2 *>(p)); }

// The 4 channels' weights, tap by tap, and bias.
template <int W>
struct Taps {
    Row w[W], b;
    __device__ __forceinline__ void load(const ConvArgs &p, int64_t c) {
        float t[kVec * W], u[kVec] = {};
        if (!p.weights_aligned) {
#pragma unroll
            for (int i = 0; i < kVec * W; ++i) t[i] = load_scalar(p.weight, c * W + i, p.weight_dtype);
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (p.bias) u[i] = load_scalar(p.bias, c + i, p.weight_dtype);
        } else if (p.weight_dtype == 1) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(p.weight) + c * W) + i);
                t[4 * i] = bf16_lo(v.x); t[4 * i + 1] = bf16_hi(v.x);
                t[4 * i + 2] = bf16_lo(v.y); t[4 * i + 3] = bf16_hi(v.y);
            }
            if (p.bias) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(p.bias) + c));
                u[0] = bf16_lo(v.x); u[1] = bf16_hi(v.x); u[2] = bf16_lo(v.y); u[3] = bf16_hi(v.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p.weight) + c * W) + i);
                t[4 * i] = v.x; t[4 * i + 1] = v.y; t[4 * i + 2] = v.z; t[4 * i + 3] = v.w;
            }
            if (p.bias) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p.bias) + c));
                u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
            }
        }
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) w[k].v[e] = f2(t[(2 * e) * W + k], t[(2 * e + 1) * W + k]);
        b.v[0] = f2(u[0], u[1]);
        b.v[1] = f2(u[2], u[3]);
    }
};

// One output row's 4 channels from the window (win[0] oldest) and the current row.
template <int W>
__device__ __forceinline__ uint2 conv_row(const Taps<W> &k, const Row (&win)[W - 1], const Row &x, bool silu) {
    uint32_t r[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint64_t acc = k.b.v[e];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) acc = fma_f2(k.w[i].v[e], win[i].v[e], acc);
        acc = fma_f2(k.w[W - 1].v[e], x.v[e], acc);
        float y0, y1;
        unf2(acc, y0, y1);
        if (silu) {
            y0 = silu_approx(y0);
            y1 = silu_approx(y1);
        }
        r[e] = pack_bf16x2(y0, y1);
    }
    return make_uint2(r[0], r[1]);
}

// Where channel c goes: the output tensor that holds it, as a pointer to its first row and
// the row's width.
__device__ __forceinline__ __nv_bfloat16 *out_of(const ConvArgs &p, int64_t c, int64_t &width) {
    int64_t first = 0;
#pragma unroll
    for (int j = 0; j < kConvMaxOutputs - 1; ++j) {
        if (j + 1 >= p.num_outputs || c < first + p.out_width[j]) {
            width = p.out_width[j];
            return static_cast<__nv_bfloat16 *>(p.out[j]) + (c - first);
        }
        first += p.out_width[j];
    }
    width = p.out_width[kConvMaxOutputs - 1];
    return static_cast<__nv_bfloat16 *>(p.out[kConvMaxOutputs - 1]) + (c - first);
}

template <int W>
__global__ void __launch_bounds__(kConvThreads)
conv_prefill_kernel(const ConvArgs p, int run, int64_t runs) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kConvThreads + threadIdx.x;
    const int64_t groups = p.channels / kVec;
    const int64_t tile = id / groups, c = (id - tile * groups) * kVec;
    const auto *x = static_cast<const __nv_bfloat16 *>(p.x) + c;
    const auto *state = p.state ? static_cast<const __nv_bfloat16 *>(p.state) + c : nullptr;
    const int64_t T = p.rows, N = p.num_seqs, C = p.channels;
    const int32_t *cu = p.cu_seqlens;
    if (tile >= runs) {
        // The new state of sequence n: rows [len, len + W - 1) of [state; x].
        const int64_t n = tile - runs;
        if (n >= N) return;
        if (c == 0) check_seq_bounds(cu, n, N, T, p.status);
        int64_t s0 = cu[n], s1 = cu[n + 1];
        s0 = s0 < 0 ? 0 : (s0 > T ? T : s0);
        s1 = s1 < s0 ? s0 : (s1 > T ? T : s1);
        auto *dst = static_cast<__nv_bfloat16 *>(p.new_state) + n * (W - 1) * C + c;
#pragma unroll
        for (int r = 0; r < W - 1; ++r) {
            const int64_t e = s1 - s0 + r;
            uint2 v = make_uint2(0, 0);
            if (e >= W - 1) v = load_row(x + (s0 + e - (W - 1)) * p.x_stride);
            else if (state) v = load_row(state + (n * (W - 1) + e) * C);
            *reinterpret_cast<uint2 *>(dst + r * C) = v;
        }
        return;
    }
    const int t0 = static_cast<int>(tile * run);
    const int t1 = static_cast<int>(t0 + run < T ? t0 + run : T);
    __shared__ uint2 ring[kBatches * kBatchRows][kConvThreads];
    const uint32_t slot0 = msync::smem_addr(&ring[0][threadIdx.x]);
    const __nv_bfloat16 *ahead = x + t0 * p.x_stride;      // the next row to copy, row t0 + copied
    int copied = 0;
    auto copy_batch = [&]() {
        const int rows = t1 - t0 - copied;
        const uint32_t to = slot0 + (copied % (kBatches * kBatchRows)) * static_cast<uint32_t>(sizeof(ring[0]));
#pragma unroll
        for (int u = 0; u < kBatchRows; ++u) {
            if (u < rows) copy_row(to + u * static_cast<uint32_t>(sizeof(ring[0])), ahead);
            ahead += p.x_stride;
        }
        copied += kBatchRows;
        msync::cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kBatches - 1; ++i) copy_batch();
    Taps<W> taps;
    taps.load(p, c);
    int64_t width;
    __nv_bfloat16 *out = out_of(p, c, width);
    out += t0 * width;
    // The sequence of token t0: the last one that starts at or before it.
    int64_t n = 0;
    for (int64_t hi = N - 1; n < hi;) {
        const int64_t mid = (n + hi + 1) >> 1;
        if (cu[mid] <= t0) n = mid;
        else hi = mid - 1;
    }
    int s0 = cu[n];
    s0 = s0 < 0 ? 0 : (s0 > t0 ? t0 : s0);
    int next = n + 1 < N ? cu[n + 1] : 0x7fffffff;
    const int end = cu[N] < t1 ? cu[N] : t1;            // rows behind the last sequence stay as they are
    // the rows in front of token t of sequence n that starts at s0
    Row win[W - 1];
    auto window = [&](int t) {
#pragma unroll
        for (int i = 0; i < W - 1; ++i) {
            const int back = W - 1 - i, at = t - back - s0;
            uint2 v = make_uint2(0, 0);
            if (at >= 0) v = load_row(x + (t - back) * p.x_stride);
            else if (state) v = load_row(state + (n * (W - 1) + (W - 1) + at) * C);
            win[i] = unpack_row(v);
        }
    };
    auto put_row = [&](uint2 w) {
        const Row cur = unpack_row(w);
        *reinterpret_cast<uint2 *>(out) = conv_row<W>(taps, win, cur, p.silu);
        out += width;
#pragma unroll
        for (int i = 0; i + 1 < W - 1; ++i) win[i] = win[i + 1];
        win[W - 2] = cur;
    };
    window(t0);
    for (int t = t0; t < end; t += kBatchRows) {
        copy_batch();                               // (into the batch read last)
        msync::cp_async_wait<kBatches - 1>();
        const uint2(*rows)[kConvThreads] = ring + (t - t0) % (kBatches * kBatchRows);
        if (end - t >= kBatchRows && next - t >= kBatchRows) {
            // whole batches inside a sequence, nearly all of them: nothing to check per row
#pragma unroll
            for (int u = 0; u < kBatchRows; ++u) put_row(rows[u][threadIdx.x]);
        } else {
#pragma unroll 1
            for (int u = 0; u < kBatchRows && t + u < end; ++u) {
                if (t + u >= next) {       // the next sequence that has tokens starts here
                    do {
                        ++n;
                        next = n + 1 < N ? cu[n + 1] : 0x7fffffff;
                    } while (t + u >= next);
                    s0 = t + u;
                    window(t + u);
                }
                put_row(rows[u][threadIdx.x]);
            }
        }
    }
    msync::cp_async_wait<0>();
}

// One token of each sequence; new_state may be state (a thread reads its own words of all
// rows before it writes any).
template <int W>
__global__ void __launch_bounds__(kConvThreads)
conv_decode_kernel(const ConvArgs p, int run, int64_t runs) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * kConvThreads + threadIdx.x;
    const int64_t groups = p.channels / kVec, C = p.channels;
    const int64_t tile = id / groups, c = (id - tile * groups) * kVec;
    if (tile >= runs) return;
    const auto *x = static_cast<const __nv_bfloat16 *>(p.x) + c;
    const auto *state = static_cast<const __nv_bfloat16 *>(p.state);
    auto *new_state = static_cast<__nv_bfloat16 *>(p.new_state);
    Taps<W> taps;
    taps.load(p, c);
    int64_t width;
    __nv_bfloat16 *out = out_of(p, c, width);
    const int64_t b1 = (tile + 1) * run < p.rows ? (tile + 1) * run : p.rows;
    for (int64_t b = tile * run; b < b1; ++b) {
        uint2 raw[W];
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            raw[i] = state ? *reinterpret_cast<const uint2 *>(state + (b * (W - 1) + i) * C + c) : make_uint2(0, 0);
        raw[W - 1] = load_row(x + b * p.x_stride);
        Row win[W - 1];
#pragma unroll
        for (int i = 0; i < W - 1; ++i) win[i] = unpack_row(raw[i]);
        *reinterpret_cast<uint2 *>(out + b * width) = conv_row<W>(taps, win, unpack_row(raw[W - 1]), p.silu);
#pragma unroll
        for (int i = 0; i < W - 1; ++i)
            *reinterpret_cast<uint2 *>(new_state + (b * (W - 1) + i) * C + c) = raw[i + 1];
    }
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    return sms;
}

// Rows per thread: the longest run (less overlap, the weights read less often) that still
// gives every SM `want` threads.
int pick_run(int64_t rows, int64_t groups, int longest, int shortest) {
    const int64_t want = static_cast<int64_t>(sm_count()) * 1024;
    int run = longest;
    while (run > shortest && ((rows + run - 1) / run) * groups < want) run /= 2;
    return run;
}

template <typename F>
cudaError_t launch_flat(F kernel, const ConvArgs &p, int run, int64_t runs, int64_t tiles, cudaStream_t stream) {
    const int64_t threads = tiles * (p.channels / kVec);
    const int64_t blocks = (threads + kConvThreads - 1) / kConvThreads;
    if (blocks > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    kernel<<<static_cast<unsigned>(blocks), kConvThreads, 0, stream>>>(p, run, runs);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_conv_prefill(const ConvArgs &p, cudaStream_t stream) {
    const int run = pick_run(p.rows, p.channels / kVec, 64, kBatchRows);
    const int64_t runs = (p.rows + run - 1) / run, tiles = runs + p.num_seqs;
    switch (p.width) {
        case 2: return launch_flat(conv_prefill_kernel<2>, p, run, runs, tiles, stream);
        case 3: return launch_flat(conv_prefill_kernel<3>, p, run, runs, tiles, stream);
        default: return launch_flat(conv_prefill_kernel<4>, p, run, runs, tiles, stream);
    }
}

cudaError_t launch_conv_decode(const ConvArgs &p, cudaStream_t stream) {
    const int run = pick_run(p.rows, p.channels / kVec, 4, 1);
    const int64_t runs = (p.rows + run - 1) / run;
    switch (p.width) {
        case 2: return launch_flat(conv_decode_kernel<2>, p, run, runs, runs, stream);
        case 3: return launch_flat(conv_decode_kernel<3>, p, run, runs, runs, stream);
        default: return launch_flat(conv_decode_kernel<4>, p, run, runs, runs, stream);
    }
}

}  // namespace gdn
