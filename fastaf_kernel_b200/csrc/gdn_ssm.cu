// gdn_ssm.cu -- the selective scan on the CUDA cores: single-token decode, and the
// token-serial prefill for very short prompts (formulas in gdn_ssm_common.cuh).
//
// Decode is HBM-bound: 8 bytes of state traffic per state element against 5 flops.  As in
// gdn_decode.cu every 8 consecutive lanes own one 512-byte state row, lane j holding the
// four float4 at columns 4j + 32m, so a warp-wide load covers four full 128-byte lines;
// each row is read once and written once.  512 sequences x 32 heads of 128: 317 us, 6.8 TB/s;
// 4 sequences: 4.8 us, which is latency (16.9 MB would take 2.6).
//
// The token-serial prefill takes about 3 us a token where every SM has more CTAs than fit (a
// CTA's tokens depend on each other: the row sums' shuffles and the next token's loads are its
// latency), so it serves prompts too short for a 64-token chunk: 16 sequences x 4 tokens, 32
// heads of 128, 26 us, and 41 in chunks.
#include "gdn_ssm_common.cuh"

namespace gdn {

namespace {

constexpr int kSsmThreads = 256;                 // 32 rows per pass (8 lanes per row)
constexpr int kSsmRowsPerPass = kSsmThreads / 8;

// This lane's 16 columns of a 128-element bf16 row.
__device__ __forceinline__ void load_cols(const void *base, int64_t at, int lane8, uint2 (&r)[4]) {
    const uint2 *q = reinterpret_cast<const uint2 *>(static_cast<const __nv_bfloat16 *>(base) + at);
#pragma unroll
    for (int m = 0; m < 4; ++m) r[m] = __ldg(q + lane8 + 8 * m);
}
__device__ __forceinline__ void unpack_cols(const uint2 (&r)[4], float (&f)[16]) {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        f[4 * m + 0] = bf16_lo(r[m].x); f[4 * m + 1] = bf16_hi(r[m].x);
        f[4 * m + 2] = bf16_lo(r[m].y); f[4 * m + 3] = bf16_hi(r[m].y);
    }
}
__device__ __forceinline__ float sum8(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    return v;
}
__device__ __forceinline__ float bf16_at(const void *p, int64_t i) {
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// y of one row, gated and rounded.
__device__ __forceinline__ void store_y(const SsmArgs &p, int64_t row, int h, int r, float y, float x, float D) {
    y = fmaf(D, x, y);
    if (p.z) y *= silu_approx(bf16_at(p.z, row * p.z_stride + h * p.head_size + r));
    static_cast<__nv_bfloat16 *>(p.out)[(row * p.heads + h) * p.head_size + r] = __float2bfloat16_rn(y);
}

template <int ROWS_PER_THREAD>
__global__ void __launch_bounds__(kSsmThreads, 3) ssm_decode_kernel(const SsmArgs p) {
    constexpr int kRowsPerCta = kSsmRowsPerPass * ROWS_PER_THREAD;
    const int ctas_per_head = p.head_size / kRowsPerCta;
    const int64_t bh = blockIdx.x / ctas_per_head;
    const int64_t b = bh / p.heads;
    const int h = static_cast<int>(bh % p.heads), g = h / (p.heads / p.groups);
    const int lane8 = threadIdx.x & 7;
    const int row0 = static_cast<int>(blockIdx.x % ctas_per_head) * kRowsPerCta + (threadIdx.x >> 3);
    const int64_t base = bh * p.head_size * kSsmState;

    float s[ROWS_PER_THREAD][16];
    // Issue every state load of this thread before any arithmetic.
#pragma unroll
    for (int r = 0; r < ROWS_PER_THREAD; ++r) {
        const float4 *sp = reinterpret_cast<const float4 *>(p.state + base + (row0 + r * kSsmRowsPerPass) * kSsmState);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float4 v = p.state ? ld_stream(sp + lane8 + 8 * m) : make_float4(0.f, 0.f, 0.f, 0.f);
            s[r][4 * m + 0] = v.x; s[r][4 * m + 1] = v.y;
            s[r][4 * m + 2] = v.z; s[r][4 * m + 3] = v.w;
        }
    }
    uint2 raw[4];
    float Bf[16], Cf[16];
    load_cols(p.B, b * p.B_stride + g * kSsmState, lane8, raw);
    unpack_cols(raw, Bf);
    load_cols(p.C, b * p.C_stride + g * kSsmState, lane8, raw);
    unpack_cols(raw, Cf);
    const float dt = ssm_step(p, b, h);
    const float decay = expf(-ssm_rate(load_scalar(p.A_log, h, p.param_dtype)) * dt);
    const float D = p.D ? load_scalar(p.D, h, p.param_dtype) : 0.0f;

#pragma unroll
    for (int r = 0; r < ROWS_PER_THREAD; ++r) {
        const int row = row0 + r * kSsmRowsPerPass;
        const float x = bf16_at(p.x, b * p.x_stride + h * p.head_size + row);
        const float u = dt * x;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[r][i] = fmaf(s[r][i], decay, u * Bf[i]);
            y = fmaf(s[r][i], Cf[i], y);
        }
        float4 *dp = reinterpret_cast<float4 *>(p.new_state + base + row * kSsmState);
#pragma unroll
        for (int m = 0; m < 4; ++m)
            st_stream(dp + lane8 + 8 * m, make_float4(s[r][4 * m], s[r][4 * m + 1], s[r][4 * m + 2], s[r][4 * m + 3]));
        y = sum8(y);
        if (lane8 == 0) store_y(p, b, h, row, y, x, D);
    }
}

// One CTA per (sequence, head, 32 state rows), the state in registers for the whole
// sequence; B, C, x and the gates of a token are fetched while the previous one is used.
__global__ void __launch_bounds__(kSsmThreads) ssm_recurrent_kernel(const SsmArgs p) {
    const int slabs = p.head_size / kSsmRowsPerPass;
    const int64_t nh = blockIdx.x / slabs;
    const int64_t n = nh / p.heads;
    const int h = static_cast<int>(nh % p.heads), g = h / (p.heads / p.groups);
    const int lane = threadIdx.x & 31, lane8 = threadIdx.x & 7;
    const int row = static_cast<int>(blockIdx.x % slabs) * kSsmRowsPerPass + (threadIdx.x >> 3);
    const int64_t T = p.rows;
    if (threadIdx.x == 0 && blockIdx.x % slabs == 0 && h == 0) check_seq_bounds(p.cu_seqlens, n, p.num_seqs, T, p.status);
    int64_t s0 = p.cu_seqlens[n], s1 = p.cu_seqlens[n + 1];
    s0 = s0 < 0 ? 0 : (s0 > T ? T : s0);
    s1 = s1 < s0 ? s0 : (s1 > T ? T : s1);

    const int64_t at = (nh * p.head_size + row) * kSsmState;
    float s[16];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const float4 v = p.state ? ld_stream(reinterpret_cast<const float4 *>(p.state + at) + lane8 + 8 * m)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
        s[4 * m + 0] = v.x; s[4 * m + 1] = v.y;
        s[4 * m + 2] = v.z; s[4 * m + 3] = v.w;
    }
    const float negA = -ssm_rate(load_scalar(p.A_log, h, p.param_dtype));
    const float D = p.D ? load_scalar(p.D, h, p.param_dtype) : 0.0f;

    uint2 rb[4], rc[4];
    float x = 0.0f, dts = 0.0f;
    auto fetch = [&](int64_t t) {
        load_cols(p.B, t * p.B_stride + g * kSsmState, lane8, rb);
        load_cols(p.C, t * p.C_stride + g * kSsmState, lane8, rc);
        x = bf16_at(p.x, t * p.x_stride + h * p.head_size + row);
    };
    if (s0 < s1) fetch(s0);
    for (int64_t t = s0; t < s1; ++t) {
        const int k = static_cast<int>((t - s0) & 31);
        if (k == 0) dts = t + lane < s1 ? ssm_step(p, t + lane, h) : 0.0f;   // 32 tokens' steps, one per lane
        const float dt = __shfl_sync(0xffffffffu, dts, k);
        const float decay = expf(negA * dt);
        float Bf[16], Cf[16];
        unpack_cols(rb, Bf);
        unpack_cols(rc, Cf);
        const float xt = x, u = dt * x;
        if (t + 1 < s1) fetch(t + 1);
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = fmaf(s[i], decay, u * Bf[i]);
            y = fmaf(s[i], Cf[i], y);
        }
        y = sum8(y);
        if (lane8 == 0) store_y(p, t, h, row, y, xt, D);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
        st_stream(reinterpret_cast<float4 *>(p.new_state + at) + lane8 + 8 * m,
                  make_float4(s[4 * m], s[4 * m + 1], s[4 * m + 2], s[4 * m + 3]));
}

}  // namespace

cudaError_t launch_ssm_decode(const SsmArgs &p, cudaStream_t stream) {
    const int64_t heads = p.rows * p.heads;
    if (heads == 0) return cudaSuccess;
    // Fewer rows per CTA when there is little state, so small batches still spread over
    // all SMs (the rule of the gated delta rule's decode kernel).
    const int rows_per_thread = heads * p.head_size >= 2048 * 128 ? 2 : 1;
    const int64_t ctas = heads * (p.head_size / (kSsmRowsPerPass * rows_per_thread));
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    if (rows_per_thread == 2) ssm_decode_kernel<2><<<static_cast<unsigned>(ctas), kSsmThreads, 0, stream>>>(p);
    else ssm_decode_kernel<1><<<static_cast<unsigned>(ctas), kSsmThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_ssm_prefill_recurrent(const SsmArgs &p, cudaStream_t stream) {
    const int64_t ctas = p.num_seqs * p.heads * (p.head_size / kSsmRowsPerPass);
    if (ctas == 0) return cudaSuccess;
    if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
    ssm_recurrent_kernel<<<static_cast<unsigned>(ctas), kSsmThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace gdn
