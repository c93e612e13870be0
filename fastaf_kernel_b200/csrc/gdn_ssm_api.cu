// gdn_ssm_api.cu -- the C ABI of the state space layer's operators (include/gdn_b200.h):
// the short causal convolution and the selective scan.  Validates arguments on the host,
// selects the kernel and launches it on the caller's stream; never synchronizes.
#include <cstdarg>
#include <cstdio>

#include "gdn_b200.h"
#include "gdn_common.cuh"
#include "gdn_launch.h"

namespace {

constexpr int64_t kMaxStride = 0x7fffffff;
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 256;      // (a run behind the last row still counts in 32 bits)
// The tensor-core scan takes a 64-token chunk of every sequence however few tokens it has, the
// token-serial one its tokens one after the other: with 32 heads of 128, 16 sequences of 4
// tokens 41 and 26 us, of 8 tokens 42 and 39, of 16 tokens 43 and 67.
constexpr int64_t kAutoTcMinTokens = 64;
constexpr int64_t kAutoTcMinPerSeq = 8;

int fail(int code, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    gdn::set_last_error(buf);
    return code;
}

int cuda_status(cudaError_t e, const char *what) {
    if (e == cudaSuccess) return GDN_OK;
    return fail(GDN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool ranges_overlap(const void *a, size_t na, const void *b, size_t nb) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

// What a call reads: `rows` rows of `width` bytes, `stride` bytes apart; or what it writes, in one
// row.  No address or no rows: nothing.
struct Span {
    const char *name;
    const void *at;
    int64_t rows, stride, width;
};
Span whole(const char *name, const void *at, int64_t bytes) { return {name, at, bytes > 0, bytes, bytes}; }

bool overlap(const Span &in, const Span &out) {
    if (!in.at || in.rows <= 0 || !out.at || out.rows <= 0) return false;
    const auto p = reinterpret_cast<uintptr_t>(in.at), o = reinterpret_cast<uintptr_t>(out.at);
    // the first row that does not end in front of the destination starts in front of its end?
    const uintptr_t k = p + in.width > o ? 0 : (o - p - in.width) / in.stride + 1;
    return k < static_cast<uintptr_t>(in.rows) && p + k * in.stride < o + out.width;
}

// Threads write what others have yet to read, or write too, where a destination overlaps an input
// or another destination.  (state and new_state, which may be one for single tokens, are checked
// by themselves.)
int refuse_overlaps(const Span *in, int num_in, const Span *out, int num_out) {
    for (int j = 0; j < num_out; ++j) {
        for (int i = 0; i < num_in; ++i)
            if (overlap(in[i], out[j]))
                return fail(GDN_ERR_INVALID_ARGUMENT, "%s must not overlap %s", out[j].name, in[i].name);
        for (int i = 0; i < j; ++i)
            if (overlap(out[i], out[j]))
                return fail(GDN_ERR_INVALID_ARGUMENT, "%s and %s must not overlap", out[j].name, out[i].name);
    }
    return GDN_OK;
}

int64_t size_of(int dtype) { return dtype == GDN_DTYPE_F32 ? 4 : 2; }

bool known_dtype(int d) { return d == GDN_DTYPE_F32 || d == GDN_DTYPE_BF16; }

// A row stride in elements: 0 stands for packed rows of `width`; anything else has to hold
// them.  Returns the stride, or -1.
int64_t row_stride(int64_t given, int64_t width) {
    if (given == 0) return width;
    return given >= width && given <= kMaxStride ? given : -1;
}

// The arguments prefill and decode of the convolution share, into `p`.
int conv_args(gdn::ConvArgs &p, const void *x, int64_t x_row_stride, const void *weight, const void *bias,
              int weight_dtype, const void *state, const int32_t *cu_seqlens, int64_t num_seqs, int64_t rows,
              int64_t channels, int width, int activation, void *const *outputs, const int64_t *output_widths, int num_outputs, void *new_state) {
    gdn::set_last_error("");
    if (width < 2 || width > 4) return fail(GDN_ERR_UNSUPPORTED, "width=%d is not supported (2, 3 or 4)", width);
    if (channels <= 0 || channels % 8 != 0 || channels > kMaxStride)
        return fail(GDN_ERR_INVALID_ARGUMENT, "channels=%lld must be a positive multiple of 8", (long long)channels);
    if (!known_dtype(weight_dtype)) return fail(GDN_ERR_INVALID_ARGUMENT, "unknown weight_dtype %d", weight_dtype);
    if (activation != GDN_ACTIVATION_NONE && activation != GDN_ACTIVATION_SILU)
        return fail(GDN_ERR_INVALID_ARGUMENT, "unknown activation %d", activation);
    if (rows < 0 || rows >= kMaxRows || num_seqs < 0 || num_seqs >= kMaxRows)
        return fail(GDN_ERR_INVALID_ARGUMENT, "tokens and sequences must be in [0, 2^31 - 256)");
    const int64_t xs = row_stride(x_row_stride, channels);
    if (xs < 0 || xs % 8 != 0)
        return fail(GDN_ERR_INVALID_ARGUMENT, "x row stride %lld must be 0 or a multiple of 8 in [channels=%lld, 2^31)",
                    (long long)x_row_stride, (long long)channels);
    if (num_outputs < 1 || num_outputs > gdn::kConvMaxOutputs || !outputs || !output_widths)
        return fail(GDN_ERR_INVALID_ARGUMENT, "num_outputs=%d must be 1 to %d, with their addresses and widths",
                    num_outputs, gdn::kConvMaxOutputs);
    int64_t sum = 0;
    for (int j = 0; j < num_outputs; ++j) {
        if (output_widths[j] <= 0 || output_widths[j] % 8 != 0 || output_widths[j] > channels)
            return fail(GDN_ERR_INVALID_ARGUMENT, "output width %lld must be a positive multiple of 8, at most channels",
                        (long long)output_widths[j]);
        sum += output_widths[j];
        p.out[j] = outputs[j];
        p.out_width[j] = output_widths[j];
    }
    if (sum != channels)
        return fail(GDN_ERR_INVALID_ARGUMENT, "the output widths add up to %lld, not to channels=%lld", (long long)sum,
                    (long long)channels);
    if (num_seqs == 0) return GDN_OK;
    if (!weight || !new_state) return fail(GDN_ERR_INVALID_ARGUMENT, "null weight or new_state");
    if (!aligned16(state) || !aligned16(new_state))
        return fail(GDN_ERR_INVALID_ARGUMENT, "state and new_state must be 16-byte aligned");
    if (rows > 0) {
        if (!x || !aligned16(x)) return fail(GDN_ERR_INVALID_ARGUMENT, "x must be a 16-byte aligned address");
        for (int j = 0; j < num_outputs; ++j)
            if (!outputs[j] || !aligned16(outputs[j]))
                return fail(GDN_ERR_INVALID_ARGUMENT, "outputs must be 16-byte aligned addresses");
    }
    const int64_t state_bytes = num_seqs * (width - 1) * channels * 2;
    const Span in[] = {{"x", x, rows, xs * 2, channels * 2},
                       whole("weight", weight, channels * width * size_of(weight_dtype)),
                       whole("bias", bias, channels * size_of(weight_dtype)),
                       whole("cu_seqlens", cu_seqlens, (num_seqs + 1) * 4),
                       whole("state", state, state_bytes)};
    Span out[gdn::kConvMaxOutputs];
    for (int j = 0; j < num_outputs; ++j) out[j] = whole("output", outputs[j], rows * output_widths[j] * 2);
    int rc = refuse_overlaps(in, 5, out, num_outputs);
    if (rc != GDN_OK) return rc;
    const Span kept = whole("new_state", new_state, state_bytes);
    if ((rc = refuse_overlaps(in, 4, &kept, 1)) != GDN_OK || (rc = refuse_overlaps(out, num_outputs, &kept, 1)) != GDN_OK)
        return rc;
    p.x = x;
    p.x_stride = xs;
    p.weight = weight;
    p.bias = bias;
    p.weight_dtype = weight_dtype;
    p.weights_aligned = aligned16(weight) && aligned16(bias);
    p.state = state;
    p.num_seqs = num_seqs;
    p.rows = rows;
    p.channels = channels;
    p.width = width;
    p.silu = activation == GDN_ACTIVATION_SILU;
    p.num_outputs = num_outputs;
    p.new_state = new_state;
    return GDN_OK;
}

size_t conv_state_bytes(const gdn::ConvArgs &p) {
    return static_cast<size_t>(p.num_seqs) * (p.width - 1) * p.channels * 2;
}

// The arguments prefill and decode of the scan share, into `p`.
int ssm_args(gdn::SsmArgs &p, const void *x, int64_t x_row_stride, const void *dt, int64_t dt_row_stride,
             const void *A_log, const void *B, int64_t B_row_stride, const void *C, int64_t C_row_stride, const void *D,
             const void *dt_bias, const void *z, int64_t z_row_stride, const float *state, const int32_t *cu_seqlens,
             int64_t num_seqs, int64_t rows, int num_heads, int num_groups, int head_size, int state_size, int dt_dtype, int param_dtype,
             void *output, float *new_state) {
    gdn::set_last_error("");
    if (state_size != 128) return fail(GDN_ERR_UNSUPPORTED, "state_size=%d is not supported (only 128)", state_size);
    if (head_size != 64 && head_size != 128)
        return fail(GDN_ERR_UNSUPPORTED, "head_size=%d is not supported (64 or 128)", head_size);
    if (num_heads <= 0 || num_groups <= 0 || num_heads % num_groups != 0 || num_heads > (1 << 20))
        return fail(GDN_ERR_INVALID_ARGUMENT, "num_heads=%d must be a positive multiple of num_groups=%d", num_heads,
                    num_groups);
    if (!known_dtype(dt_dtype) || !known_dtype(param_dtype))
        return fail(GDN_ERR_INVALID_ARGUMENT, "unknown dtype code (dt %d, params %d)", dt_dtype, param_dtype);
    if (rows < 0 || rows >= kMaxRows || num_seqs < 0 || num_seqs >= kMaxRows)
        return fail(GDN_ERR_INVALID_ARGUMENT, "tokens and sequences must be in [0, 2^31 - 256)");
    const int64_t wide = static_cast<int64_t>(num_heads) * head_size, bc = static_cast<int64_t>(num_groups) * 128;
    p.x_stride = row_stride(x_row_stride, wide);
    p.z_stride = row_stride(z_row_stride, wide);
    p.B_stride = row_stride(B_row_stride, bc);
    p.C_stride = row_stride(C_row_stride, bc);
    p.dt_stride = row_stride(dt_row_stride, num_heads);
    if (p.x_stride < 0 || p.z_stride < 0 || p.B_stride < 0 || p.C_stride < 0 || p.dt_stride < 0)
        return fail(GDN_ERR_INVALID_ARGUMENT, "row strides must be 0 or in [row width, 2^31)");
    if (p.x_stride % 8 || p.z_stride % 8 || p.B_stride % 8 || p.C_stride % 8)
        return fail(GDN_ERR_INVALID_ARGUMENT, "row strides of x, z, B and C must be multiples of 8");
    if (num_seqs == 0) return GDN_OK;
    if (!A_log || !new_state) return fail(GDN_ERR_INVALID_ARGUMENT, "null A_log or new_state");
    if (!aligned16(state) || !aligned16(new_state))
        return fail(GDN_ERR_INVALID_ARGUMENT, "state and new_state must be 16-byte aligned");
    if (rows > 0) {
        if (!x || !dt || !B || !C || !output) return fail(GDN_ERR_INVALID_ARGUMENT, "null x, dt, B, C or output");
        if (!aligned16(x) || !aligned16(B) || !aligned16(C) || !aligned16(z) || !aligned16(output))
            return fail(GDN_ERR_INVALID_ARGUMENT, "x, B, C, z and output must be 16-byte aligned");
    }
    const int64_t state_bytes = num_seqs * num_heads * head_size * 128 * 4, each = size_of(dt_dtype);
    const int64_t params = num_heads * size_of(param_dtype);
    const Span in[] = {{"x", x, rows, p.x_stride * 2, wide * 2},
                       {"dt", dt, rows, p.dt_stride * each, num_heads * each},
                       {"B", B, rows, p.B_stride * 2, bc * 2},
                       {"C", C, rows, p.C_stride * 2, bc * 2},
                       {"z", z, rows, p.z_stride * 2, wide * 2},
                       whole("A_log", A_log, params),
                       whole("D", D, params),
                       whole("dt_bias", dt_bias, params),
                       whole("cu_seqlens", cu_seqlens, (num_seqs + 1) * 4),
                       whole("state", state, state_bytes)};
    const Span out = whole("output", output, rows * wide * 2), kept = whole("new_state", new_state, state_bytes);
    int rc = refuse_overlaps(in, 10, &out, 1);
    if (rc != GDN_OK || (rc = refuse_overlaps(in, 9, &kept, 1)) != GDN_OK || (rc = refuse_overlaps(&out, 1, &kept, 1)) != GDN_OK)
        return rc;
    p.x = x;
    p.dt = dt;
    p.B = B;
    p.C = C;
    p.z = z;
    p.A_log = A_log;
    p.D = D;
    p.dt_bias = dt_bias;
    p.dt_dtype = dt_dtype;
    p.param_dtype = param_dtype;
    p.state = state;
    p.num_seqs = num_seqs;
    p.rows = rows;
    p.heads = num_heads;
    p.groups = num_groups;
    p.head_size = head_size;
    p.out = output;
    p.new_state = new_state;
    return GDN_OK;
}

size_t ssm_state_bytes(const gdn::SsmArgs &p) {
    return static_cast<size_t>(p.num_seqs) * p.heads * p.head_size * 128 * 4;
}

}  // namespace

extern "C" {

int gdn_conv_prefill(const void *x, int64_t x_row_stride, const void *weight, const void *bias, int weight_dtype,
                     const void *state, const int32_t *cu_seqlens, int64_t num_seqs, int64_t total_tokens,
                     int64_t channels, int width, int activation, void *const *outputs, const int64_t *output_widths,
                     int num_outputs, void *new_state, void *stream) {
    gdn::ConvArgs p{};
    const int rc = conv_args(p, x, x_row_stride, weight, bias, weight_dtype, state, cu_seqlens, num_seqs, total_tokens,
                             channels, width, activation, outputs, output_widths, num_outputs, new_state);
    if (rc != GDN_OK || num_seqs == 0) return rc;
    if (!cu_seqlens) return fail(GDN_ERR_INVALID_ARGUMENT, "null cu_seqlens");
    // (a long sequence is split over threads: its end writes what its start reads)
    if (state && ranges_overlap(state, conv_state_bytes(p), new_state, conv_state_bytes(p)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "prefill new_state must not overlap state");
    p.cu_seqlens = cu_seqlens;
    p.status = gdn::device_status_word();
    return cuda_status(gdn::launch_conv_prefill(p, static_cast<cudaStream_t>(stream)), "gdn_conv_prefill launch");
}

int gdn_conv_decode(const void *x, int64_t x_row_stride, const void *weight, const void *bias, int weight_dtype,
                    const void *state, int64_t batch, int64_t channels, int width, int activation,
                    void *const *outputs, const int64_t *output_widths, int num_outputs, void *new_state,
                    void *stream) {
    gdn::ConvArgs p{};
    const int rc = conv_args(p, x, x_row_stride, weight, bias, weight_dtype, state, nullptr, batch, batch, channels,
                             width, activation, outputs, output_widths, num_outputs, new_state);
    if (rc != GDN_OK || batch == 0) return rc;
    if (state && state != new_state && ranges_overlap(state, conv_state_bytes(p), new_state, conv_state_bytes(p)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "new_state partially overlaps state (only exact aliasing is allowed)");
    return cuda_status(gdn::launch_conv_decode(p, static_cast<cudaStream_t>(stream)), "gdn_conv_decode launch");
}

int gdn_ssm_resolve(int64_t total_tokens, int64_t num_seqs, int method) {
    if (method != GDN_PREFILL_AUTO) return method;
    // Short prompts: the token-serial kernel, which also keeps every product in fp32.
    if (total_tokens < kAutoTcMinTokens || total_tokens < kAutoTcMinPerSeq * num_seqs ||
        !gdn::ssm_prefill_tc_supported(total_tokens))
        return GDN_PREFILL_RECURRENT;
    return GDN_PREFILL_TCGEN05;
}

int gdn_ssm_prefill(const void *x, int64_t x_row_stride, const void *dt, int64_t dt_row_stride, const void *A_log,
                    const void *B, int64_t B_row_stride, const void *C, int64_t C_row_stride, const void *D,
                    const void *dt_bias, const void *z, int64_t z_row_stride, const float *state,
                    const int32_t *cu_seqlens, int64_t num_seqs, int64_t total_tokens, int num_heads, int num_groups,
                    int head_size, int state_size, int dt_dtype, int param_dtype, void *output, float *new_state,
                    int method, void *stream) {
    gdn::SsmArgs p{};
    const int rc = ssm_args(p, x, x_row_stride, dt, dt_row_stride, A_log, B, B_row_stride, C, C_row_stride, D, dt_bias,
                            z, z_row_stride, state, cu_seqlens, num_seqs, total_tokens, num_heads, num_groups,
                            head_size, state_size, dt_dtype, param_dtype, output, new_state);
    if (rc != GDN_OK) return rc;
    if (method != GDN_PREFILL_AUTO && method != GDN_PREFILL_RECURRENT && method != GDN_PREFILL_TCGEN05)
        return fail(GDN_ERR_INVALID_ARGUMENT, "unknown scan method %d", method);
    if (num_seqs == 0) return GDN_OK;
    if (!cu_seqlens) return fail(GDN_ERR_INVALID_ARGUMENT, "null cu_seqlens");
    if (state && ranges_overlap(state, ssm_state_bytes(p), new_state, ssm_state_bytes(p)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "prefill new_state must not overlap state");
    p.cu_seqlens = cu_seqlens;
    p.status = gdn::device_status_word();
    const auto s = static_cast<cudaStream_t>(stream);
    if (gdn_ssm_resolve(total_tokens, num_seqs, method) == GDN_PREFILL_TCGEN05) {
        if (!gdn::ssm_prefill_tc_supported(total_tokens))
            return fail(GDN_ERR_UNSUPPORTED, "the tcgen05 scan needs an sm_100 device and total_tokens >= 64");
        return cuda_status(gdn::launch_ssm_prefill_tc(p, s), "gdn_ssm_prefill (tcgen05) launch");
    }
    return cuda_status(gdn::launch_ssm_prefill_recurrent(p, s), "gdn_ssm_prefill (recurrent) launch");
}

int gdn_ssm_decode(const void *x, int64_t x_row_stride, const void *dt, int64_t dt_row_stride, const void *A_log,
                   const void *B, int64_t B_row_stride, const void *C, int64_t C_row_stride, const void *D,
                   const void *dt_bias, const void *z, int64_t z_row_stride, const float *state, int64_t batch,
                   int num_heads, int num_groups, int head_size, int state_size, int dt_dtype, int param_dtype,
                   void *output, float *new_state, void *stream) {
    gdn::SsmArgs p{};
    const int rc = ssm_args(p, x, x_row_stride, dt, dt_row_stride, A_log, B, B_row_stride, C, C_row_stride, D, dt_bias,
                            z, z_row_stride, state, nullptr, batch, batch, num_heads, num_groups, head_size,
                            state_size, dt_dtype, param_dtype, output, new_state);
    if (rc != GDN_OK || batch == 0) return rc;
    if (state && state != new_state && ranges_overlap(state, ssm_state_bytes(p), new_state, ssm_state_bytes(p)))
        return fail(GDN_ERR_INVALID_ARGUMENT, "new_state partially overlaps state (only exact aliasing is allowed)");
    return cuda_status(gdn::launch_ssm_decode(p, static_cast<cudaStream_t>(stream)), "gdn_ssm_decode launch");
}

}  // extern "C"
