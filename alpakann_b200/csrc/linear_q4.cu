// linear_q4.cu -- products with weights held in 4 bits.
//
// A weight W[k, n] (row-major [in, out], as linear's) is (u - 8) * s: u is its
// nibble, s the fp32 scale of its group of `group` consecutive inputs and its
// column. Eight consecutive inputs of a column share one 32-bit word, the first
// in the low bits:
//   packed [K / 8, N] int32, scales [ceil(K / group), N].
//   y[m, n] = act(sum_k x[m, k] W[k, n] + bias[n]) + residual[m, n]
#include <algorithm>

#include "common.cuh"
#include "reduce.cuh"

namespace ann {
namespace {

struct LinearQ4Args {
    const float* x;
    const uint32_t* w;
    const float* s;
    const float* bias;  // may be null
    const float* res;   // may be null
    float* y;
    int64_t x_m, x_k, w_r, w_n, s_g, s_n, b_n, r_m, r_n, y_m, y_n;
    int64_t M, K, N;
    int group, act;
};

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ANN_ACT_RELU: return v > 0.0f ? v : 0.0f;
        case ANN_ACT_SILU: return v / (1.0f + expf(-v));
        case ANN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        default: return v;
    }
}

constexpr int kThreads = 128;

// A thread per column.
__global__ void __launch_bounds__(kThreads) linear_q4_kernel(LinearQ4Args a) {
    int64_t const n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, m = blockIdx.y;
    if (n >= a.N) return;
    float const* x = a.x + m * a.x_m;
    float acc = 0.0f;
    for (int64_t k0 = 0; k0 < a.K; k0 += a.group) {
        int64_t const k1 = min(a.K, k0 + a.group);
        float sum = 0.0f;
        for (int64_t k = k0; k < k1; k += 8) {
            uint32_t const w = a.w[k / 8 * a.w_r + n * a.w_n];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                sum = fmaf(x[(k + j) * a.x_k], static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8), sum);
        }
        acc = fmaf(sum, a.s[k0 / a.group * a.s_g + n * a.s_n], acc);
    }
    if (a.bias != nullptr) acc += a.bias[n * a.b_n];
    acc = activate(acc, a.act);
    if (a.res != nullptr) acc += a.res[m * a.r_m + n * a.r_n];
    a.y[m * a.y_m + n * a.y_n] = acc;
}

struct PackArgs {
    const float* w;
    uint32_t* packed;
    float* s;
    int64_t w_k, w_n, p_r, p_n, s_g, s_n;
    int64_t K, N;
    int group;
};

// The whole number nearest to v / s (ties to even), from the exact quotient of
// two 32-bit values in 64 bits, in [-7, 7].
__device__ __forceinline__ uint32_t nibble(float v, float s) {
    if (!(s > 0.0f) || __float_as_uint(s) >= 0x7f800000u) return 8u;  // zero, NaN or infinite scale: n = 0
    double const n = fmin(fmax(rint(static_cast<double>(v) / static_cast<double>(s)), -7.0), 7.0);
    return static_cast<uint32_t>(static_cast<int>(n) + 8);
}

// A thread per column and group. Packing happens once, when weights are loaded.
__global__ void __launch_bounds__(kThreads) pack_kernel(PackArgs a) {
    int64_t const n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (n >= a.N) return;
    int64_t const groups = (a.K + a.group - 1) / a.group;
    for (int64_t g = blockIdx.y; g < groups; g += gridDim.y) {
        int64_t const k0 = g * a.group, k1 = min(a.K, k0 + a.group);
        unsigned int top = 0;  // max |w| on the bit patterns: NaN above infinity above every number
        for (int64_t k = k0; k < k1; ++k) top = max(top, __float_as_uint(a.w[k * a.w_k + n * a.w_n]) & 0x7fffffffu);
        float const s = __fdiv_rn(__uint_as_float(top), 7.0f);
        a.s[g * a.s_g + n * a.s_n] = s;
        for (int64_t k = k0; k < k1; k += 8) {
            uint32_t word = 0;
            for (int j = 0; j < 8; ++j) word |= nibble(a.w[(k + j) * a.w_k + n * a.w_n], s) << (4 * j);
            a.packed[k / 8 * a.p_r + n * a.p_n] = word;
        }
    }
}

// packed [K/8, N] and scales [ceil(K/group), N].
int check_packed(const char* what, const ann_view* p_v, const ann_view* s_v, uint32_t group, Dims& p, Dims& s) {
    ANN_TRY(to_dims(p_v, sizeof(uint32_t), what, p));
    ANN_TRY(to_dims(s_v, sizeof(float), what, s));
    if (p.rank != 2 || s.rank != 2) return fail(ANN_EINVAL, "%s expects rank-2 packed weights and scales.", what);
    if (group == 0 || group % 32 != 0 || group > (1u << 30))
        return fail(ANN_EINVAL, "%s requires a group size that is a positive multiple of 32.", what);
    if (s.ext[1] != p.ext[1] || s.ext[0] != ceil_div(8 * p.ext[0], group))
        return fail(ANN_EINVAL, "%s: scales %s do not match packed weights %s in groups of %u.", what,
                    extents_str(s).c_str(), extents_str(p).c_str(), group);
    return ANN_OK;
}

int linear_q4(ann_stream stream, const ann_view* x_v, const ann_view* p_v, const ann_view* s_v, const ann_view* b_v,
              const ann_view* r_v, const ann_view* y_v, uint32_t group, int act) {
    Dims x, p, s, b, r, y;
    ANN_TRY(to_dims(x_v, sizeof(float), "linearQ4 input", x));
    ANN_TRY(check_packed("linearQ4", p_v, s_v, group, p, s));
    ANN_TRY(to_dims(y_v, sizeof(float), "linearQ4 output", y));
    if (act < ANN_ACT_NONE || act > ANN_ACT_GELU) return fail(ANN_EINVAL, "linearQ4: unknown activation %d.", act);
    if (x.rank != 2 || y.rank != 2 || x.ext[1] != 8 * p.ext[0] || y.ext[0] != x.ext[0] || y.ext[1] != p.ext[1])
        return fail(ANN_EINVAL, "linearQ4 shape mismatch.");
    if (!writable(y)) return fail(ANN_EINVAL, "linearQ4: an output axis has a zero pitch.");
    LinearQ4Args a{};
    if (b_v != nullptr) {
        ANN_TRY(to_dims(b_v, sizeof(float), "linearQ4 bias", b));
        if (b.rank != 1 || b.ext[0] != y.ext[1]) return fail(ANN_EINVAL, "linearQ4 expects a 1D bias matching the output.");
        a.bias = static_cast<const float*>(b.data);
        a.b_n = b.str[0];
    }
    if (r_v != nullptr) {
        ANN_TRY(to_dims(r_v, sizeof(float), "linearQ4 residual", r));
        if (!same_extents(r, y)) return fail(ANN_EINVAL, "linearQ4: the residual must have the extents of the output.");
        a.res = static_cast<const float*>(r.data);
        a.r_m = r.str[0];
        a.r_n = r.str[1];
    }
    if (y.numel() == 0) return ANN_OK;
    a.x = static_cast<const float*>(x.data);
    a.w = static_cast<const uint32_t*>(p.data);
    a.s = static_cast<const float*>(s.data);
    a.y = static_cast<float*>(y.data);
    a.x_m = x.str[0], a.x_k = x.str[1];
    a.w_r = p.str[0], a.w_n = p.str[1];
    a.s_g = s.str[0], a.s_n = s.str[1];
    a.y_m = y.str[0], a.y_n = y.str[1];
    a.M = x.ext[0];
    a.K = x.ext[1];
    a.N = y.ext[1];
    a.group = static_cast<int>(group);
    a.act = act;
    if (a.M > 65535) return fail(ANN_ENOTSUP, "linearQ4: more than 65535 rows.");
    int64_t const gx = ceil_div(a.N, kThreads);
    if (gx > INT32_MAX) return fail(ANN_ENOTSUP, "linearQ4: too many columns.");
    linear_q4_kernel<<<dim3(static_cast<unsigned>(gx), static_cast<unsigned>(a.M)), kThreads, 0, as_stream(stream)>>>(a);
    return check_launch("linearQ4");
}

int pack_q4(ann_stream stream, const ann_view* w_v, const ann_view* p_v, const ann_view* s_v, uint32_t group) {
    Dims w, p, s;
    ANN_TRY(to_dims(w_v, sizeof(float), "packWeightQ4 weight", w));
    ANN_TRY(check_packed("packWeightQ4", p_v, s_v, group, p, s));
    if (w.rank != 2 || w.ext[0] != 8 * p.ext[0] || w.ext[1] != p.ext[1])
        return fail(ANN_EINVAL, "packWeightQ4: weight %s does not match packed %s (eight inputs a word).",
                    extents_str(w).c_str(), extents_str(p).c_str());
    if (!writable(p) || !writable(s)) return fail(ANN_EINVAL, "packWeightQ4: an output axis has a zero pitch.");
    if (w.numel() == 0) return ANN_OK;
    PackArgs a{static_cast<const float*>(w.data), static_cast<uint32_t*>(p.data), static_cast<float*>(s.data),
               w.str[0], w.str[1], p.str[0], p.str[1], s.str[0], s.str[1], w.ext[0], w.ext[1], static_cast<int>(group)};
    int64_t const gx = ceil_div(a.N, kThreads);
    if (gx > INT32_MAX) return fail(ANN_ENOTSUP, "packWeightQ4: too many columns.");
    dim3 const grid(static_cast<unsigned>(gx), static_cast<unsigned>(std::min<int64_t>(s.ext[0], 65535)));
    pack_kernel<<<grid, kThreads, 0, as_stream(stream)>>>(a);
    return check_launch("packWeightQ4");
}

}  // namespace
}  // namespace ann

extern "C" {

int ann_linear_q4_f32(ann_stream st, const ann_view* input, const ann_view* packed, const ann_view* scales,
                      const ann_view* bias, const ann_view* residual, const ann_view* output, uint32_t group_size,
                      int32_t act) {
    ANN_API_BEGIN
    return ann::linear_q4(st, input, packed, scales, bias, residual, output, group_size, act);
    ANN_API_END
}

int ann_pack_weight_q4_f32(ann_stream st, const ann_view* weight, const ann_view* packed, const ann_view* scales,
                           uint32_t group_size) {
    ANN_API_BEGIN
    return ann::pack_q4(st, weight, packed, scales, group_size);
    ANN_API_END
}

}  // extern "C"
