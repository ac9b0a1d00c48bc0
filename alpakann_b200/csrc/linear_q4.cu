// linear_q4.cu -- products with weights held in 4 bits.
//
// A weight W[k, n] (row-major [in, out], as linear's) is (u - 8) * s: u is its
// nibble, s the fp32 scale of its group of `group` consecutive inputs and its
// column. Eight consecutive inputs of a column share one 32-bit word, the first
// in the low bits:
//   packed [K / 8, N] int32, scales [ceil(K / group), N].
//   y[m, n] = act(sum_k x[m, k] W[k, n] + bias[n]) + residual[m, n]
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <set>

#include "common.cuh"
#include "tma.cuh"

namespace cg = cooperative_groups;

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
    int x_vec;   // eight inputs are two aligned 16-byte loads
    int splits;  // CTAs of a cluster that share the inputs
};

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ANN_ACT_RELU: return v > 0.0f ? v : 0.0f;
        case ANN_ACT_SILU: return v / (1.0f + expf(-v));
        case ANN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        default: return v;
    }
}

// The product on mma.sync.m16n8k16, transposed: 16 columns of W by 8 slots, the
// slots being the two fp16 parts (11 bits each) of up to four rows of x, so that
// one product gives both parts of four rows in the same thread and the weights
// -- whole numbers -8..7, exact in fp16 -- are converted once for all rows. Sums
// are fp32; every 32 inputs they leave the tensor core and meet their group's
// scale. The order of the summed index is free, so a lane takes the words as a
// 16-byte load gives them: eight inputs (its octet of 32) of four neighbouring
// columns, whose nibbles j and j + 4 sit 16 bits apart and become a fp16 pair with
// one mask and one addition; x is laid out to match.
//
// A CTA takes 32 CT columns, its warps (and the CTAs of a cluster) the inputs;
// partial sums meet in shared memory and, across the cluster, in the CTA that
// owns a share of the columns, which applies bias, activation and residual. One
// launch, no scratch memory, no atomics, a fixed order of sums.
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 16;
constexpr uint32_t kZeros = 0x88888888u;  // eight weights of 0

// d += a b (or d = a b), fp16 products summed in fp32.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t const*>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t w) { return *reinterpret_cast<__half2 const*>(&w); }

// A word's weights as fp16 pairs (j, j + 4), j = 0..3. 0x6400 | u is 1024 + u, and
// 1032 is taken off; with the nibble 4 bits higher it is 1024 + 16 u, of which a
// sixteenth less 72 is left. All exact.
__device__ __forceinline__ void weights_of(uint32_t w, uint32_t (&h)[4]) {
    __half2 const off = half2_of(0x64086408u), sixteenth = half2_of(0x2c002c00u), off16 = half2_of(0xd480d480u);
    uint32_t const v = w >> 8;
    h[0] = bits(__hsub2(half2_of((w & 0x000f000fu) | 0x64006400u), off));
    h[1] = bits(__hfma2(half2_of((w & 0x00f000f0u) | 0x64006400u), sixteenth, off16));
    h[2] = bits(__hsub2(half2_of((v & 0x000f000fu) | 0x64006400u), off));
    h[3] = bits(__hfma2(half2_of((v & 0x00f000f0u) | 0x64006400u), sixteenth, off16));
}

// CT: 16-byte words of columns per lane (32 CT columns a CTA); NT: slots / 8 (4 NT
// rows a CTA); VEC: words and scales of four columns are one aligned load.
template <int CT, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1) linear_q4_kernel(LinearQ4Args a) {
    constexpr int COLS = 32 * CT, ROWS = 4 * NT, ITEMS = ROWS * COLS;
    extern __shared__ __align__(16) float sums[];  // [kWarps][ROWS][COLS], then [splits][per]
    int const tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int const split = static_cast<int>(blockIdx.x) % a.splits;
    if (a.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // "this CTA runs"
    int64_t const col0 = static_cast<int64_t>(blockIdx.x / a.splits) * COLS, row0 = static_cast<int64_t>(blockIdx.y) * ROWS;
    // this warp's steps of 32 inputs
    int const steps = static_cast<int>((a.K + 31) / 32), parts = a.splits * kWarps, part = split * kWarps + warp;
    int const s0 = static_cast<int>(static_cast<int64_t>(steps) * part / parts);
    int const s1 = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / parts);
    int const octets = static_cast<int>(a.K / 8);

    auto load_w = [&](int step, uint32_t (&w)[CT][4]) {
        int const r = 4 * step + t;
        uint32_t const* p = a.w + r * a.w_r;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            int64_t const n = col0 + 32 * c + 4 * g;
            if constexpr (VEC) {
                uint4 v = make_uint4(kZeros, kZeros, kZeros, kZeros);
                if (r < octets && n < a.N) v = __ldg(reinterpret_cast<uint4 const*>(p + n));
                w[c][0] = v.x, w[c][1] = v.y, w[c][2] = v.z, w[c][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[c][e] = r < octets && n + e < a.N ? __ldg(p + (n + e) * a.w_n) : kZeros;
            }
        }
    };
    // x of slot row g / 2 (+ 4 nt): this lane's octet of a step
    auto load_x = [&](int step, int nt, float (&x)[8]) {
        int64_t const m = row0 + 4 * nt + (g >> 1), k = 32 * static_cast<int64_t>(step) + 8 * t;
        bool const in = m < a.M && k < a.K;
        float const* p = a.x + m * a.x_m + k * a.x_k;
        if (a.x_vec) {
            float4 const zero = make_float4(0.f, 0.f, 0.f, 0.f);
            float4 const u = in ? *reinterpret_cast<float4 const*>(p) : zero;
            float4 const v = in ? *reinterpret_cast<float4 const*>(p + 4) : zero;
            x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = in ? p[e * a.x_k] : 0.0f;
        }
    };

    uint32_t w[2][CT][4];
    if (s0 < s1) load_w(s0, w[0]);
    // The power of two that brings this warp's largest |x| of each row to [2^13, 2^14).
    float up[NT], down[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        unsigned int top = 0;
        for (int s = s0; s < s1; ++s) {
            float x[8];
            load_x(s, nt, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = static_cast<int>(top >> 23);
        e = e == 255 ? 140 : max(e, 15);  // NaN and infinity pass through as they are
        up[nt] = __int_as_float((267 - e) << 23);
        // slot 2t holds row t: its lane's factor
        down[nt] = __shfl_sync(0xffffffffu, __int_as_float((e - 13) << 23), 8 * t);
    }

    float acc[NT][CT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][c][e] = 0.0f;

    for (int s = s0; s < s1; s += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            int const step = s + u;
            if (step >= s1) break;
            if (step + 1 < s1) load_w(step + 1, w[u ^ 1]);
            uint32_t b[NT][4];  // pairs (j, j + 4)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float x[8];
                load_x(step, nt, x);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float const y0 = x[j] * up[nt], y1 = x[j + 4] * up[nt];
                    __half2 const hi = __floats2half2_rn(y0, y1);
                    float2 const f = __half22float2(hi);
                    __half2 const lo = __floats2half2_rn(isinf(f.x) ? 0.0f : y0 - f.x, isinf(f.y) ? 0.0f : y1 - f.y);
                    b[nt][j] = g & 1 ? bits(lo) : bits(hi);
                }
            }
            int64_t const group = 32 * static_cast<int64_t>(step) / a.group;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                int64_t const n = col0 + 32 * c + 4 * g;
                float sc[4] = {0.f, 0.f, 0.f, 0.f};
                float const* ps = a.s + group * a.s_g;
                if constexpr (VEC) {
                    if (n < a.N) {
                        float4 const v = __ldg(reinterpret_cast<float4 const*>(ps + n));
                        sc[0] = v.x, sc[1] = v.y, sc[2] = v.z, sc[3] = v.w;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n + e < a.N) sc[e] = __ldg(ps + (n + e) * a.s_n);
                }
                uint32_t h[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) weights_of(w[u][c][e], h[e]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {  // columns 4g + e, 4g + e + 1 are rows g, g + 8 of the product
                        float d[4];
                        mma_f16_first(d, h[e][0], h[e + 1][0], h[e][1], h[e + 1][1], b[nt][0], b[nt][1]);
                        mma_f16(d, h[e][2], h[e + 1][2], h[e][3], h[e + 1][3], b[nt][2], b[nt][3]);
                        acc[nt][c][e] = fmaf(d[0] + d[1], sc[e], acc[nt][c][e]);
                        acc[nt][c][e + 1] = fmaf(d[2] + d[3], sc[e + 1], acc[nt][c][e + 1]);
                    }
            }
        }
    }
    // Warps to CTA.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < CT; ++c)
            *reinterpret_cast<float4*>(sums + (warp * ROWS + 4 * nt + t) * COLS + 32 * c + 4 * g) =
                make_float4(acc[nt][c][0] * down[nt], acc[nt][c][1] * down[nt], acc[nt][c][2] * down[nt],
                            acc[nt][c][3] * down[nt]);
    __syncthreads();
    int const rows = static_cast<int>(min(static_cast<int64_t>(ROWS), a.M - row0));
    int const cols = static_cast<int>(min(static_cast<int64_t>(COLS), a.N - col0));
    auto sum_warps = [&](int i) {
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v += sums[k * ITEMS + i];
        return v;
    };
    auto store = [&](int i, float v) {
        int const r = i / COLS, c = i - r * COLS;
        if (r >= rows || c >= cols) return;
        int64_t const m = row0 + r, n = col0 + c;
        if (a.bias != nullptr) v += a.bias[n * a.b_n];
        v = activate(v, a.act);
        if (a.res != nullptr) v += a.res[m * a.r_m + n * a.r_n];
        a.y[m * a.y_m + n * a.y_n] = v;
    };
    int const items = rows * COLS;
    if (a.splits == 1) {
        for (int i = tid; i < items; i += kThreads) store(i, sum_warps(i));
        return;
    }
    // CTAs of the cluster: CTA s takes items [s * per, (s + 1) * per) of all of them.
    cg::cluster_group cluster = cg::this_cluster();
    int const per = (items + a.splits - 1) / a.splits;
    float* recv = sums + kWarps * ITEMS;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA runs
    for (int i = tid; i < items; i += kThreads) {
        int const to = i / per;
        cluster.map_shared_rank(recv, to)[split * per + i - to * per] = sum_warps(i);
    }
    cluster_sync();
    for (int i = split * per + tid; i < min(items, (split + 1) * per); i += kThreads) {
        float v = 0.0f;
        for (int k = 0; k < a.splits; ++k) v += recv[k * per + i - split * per];
        store(i, v);
    }
}

template <int CT, int NT, bool VEC>
int launch(ann_stream stream, LinearQ4Args& a) {
    constexpr int COLS = 32 * CT, ROWS = 4 * NT;
    constexpr size_t smem = sizeof(float) * ((kWarps + 1) * ROWS * COLS + kMaxCluster);
    auto const kernel = linear_q4_kernel<CT, NT, VEC>;
    static std::mutex mu;
    static std::set<int> ready;  // devices whose kernel attributes are set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "linearQ4: no CUDA device.");
    {
        std::lock_guard<std::mutex> lock(mu);
        if (ready.count(dev) == 0) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return fail(ANN_ECUDA, "linearQ4 setup: %s", cudaGetErrorString(e));
            ready.insert(dev);
        }
    }
    int64_t const tiles = ceil_div(a.N, COLS), row_tiles = ceil_div(a.M, ROWS);
    int64_t const steps = ceil_div(a.K, 32);
    int64_t const want = ceil_div(int64_t{2} * sm_count(), tiles * row_tiles);
    a.splits = static_cast<int>(std::max<int64_t>(1, std::min({want, ceil_div(steps, 2 * kWarps), int64_t{kMaxCluster}})));
    if (const char* e = std::getenv("TUNE_S")) a.splits = std::atoi(e);
    if (tiles * a.splits > INT32_MAX || row_tiles > 65535) return fail(ANN_ENOTSUP, "linearQ4: grid too large.");
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.splits), static_cast<unsigned>(row_tiles));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = as_stream(stream);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t const e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return fail(ANN_ECUDA, "linearQ4: %s", cudaGetErrorString(e));
    return check_launch("linearQ4");
}

template <int CT, int NT>
int launch_vec(ann_stream stream, LinearQ4Args& a, bool vec) {
    return vec ? launch<CT, NT, true>(stream, a) : launch<CT, NT, false>(stream, a);
}

template <int CT>
int launch_rows(ann_stream stream, LinearQ4Args& a, bool vec) {
    if (a.M <= 4) return launch_vec<CT, 1>(stream, a, vec);
    if (a.M <= 8) return launch_vec<CT, 2>(stream, a, vec);
    return launch_vec<CT, 4>(stream, a, vec);
}

constexpr int kPackThreads = 128;

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
__global__ void __launch_bounds__(kPackThreads) pack_kernel(PackArgs a) {
    int64_t const n = static_cast<int64_t>(blockIdx.x) * kPackThreads + threadIdx.x;
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
    if (x.ext[1] > INT32_MAX) return fail(ANN_ENOTSUP, "linearQ4: more than 2^31 inputs.");
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
    a.x_vec = a.x_k == 1 && a.x_m % 4 == 0 && aligned(x.data, 16);
    bool const vec = a.w_n == 1 && a.w_r % 4 == 0 && aligned(p.data, 16) && a.s_n == 1 && a.s_g % 4 == 0 &&
                     aligned(s.data, 16) && a.N % 4 == 0;
    bool const narrow = std::getenv("TUNE_C") ? std::atoi(std::getenv("TUNE_C")) == 1 : a.N * ceil_div(a.M, 16) < 2048;
    return narrow ? launch_rows<1>(stream, a, vec) : launch_rows<4>(stream, a, vec);
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
    int64_t const gx = ceil_div(a.N, kPackThreads);
    if (gx > INT32_MAX) return fail(ANN_ENOTSUP, "packWeightQ4: too many columns.");
    dim3 const grid(static_cast<unsigned>(gx), static_cast<unsigned>(std::min<int64_t>(s.ext[0], 65535)));
    pack_kernel<<<grid, kPackThreads, 0, as_stream(stream)>>>(a);
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
