// rotary.cu -- rotary positions with a position per token.
//
// For pair p of a head vector at position t, with a = t * f[p] in 64 bits,
//   (x0, x1) -> m * (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
// where the pair is (2p, 2p+1) (interleaved) or (p, p + R/2) (halves), R = 2
// len(f) elements of the head are turned and the rest pass through. With a
// negated angle the same kernel applies the transposed rotation, which is the
// gradient with respect to the input.
//
// No cos/sin table is read: the angles are formed from the position and the
// frequency, so a far or irregular position costs nothing extra and the bytes
// moved are one read and one write of q and k. The 64-bit product is what far
// positions need (position 100000 leaves 7 bits of fraction in a 32-bit
// angle); it is brought within an eighth of a turn of a whole quarter in 64 bits and only
// then rounded to the tensor's type, so fp32 takes one single-precision sincospi per pair.
// A thread forms the angles of its pairs once and walks over heads with them. Bound by
// HBM; measured: 4 x 4096 tokens, 32 + 32 heads of 128 180 us (0.92 of the bytes' time at
// the copy rate), fp64 2 x 1024 tokens, 16 + 16 heads of 64 12.1 us (0.86), 16 single
// tokens 2.9 us, a launch.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "overlap.cuh"
#include "reduce.cuh"

namespace ann {
namespace {

constexpr int kThreads = 256;
constexpr int kHeadsAtOnce = 4;  // heads whose loads are issued together

struct RotaryJob {
    const void* in;
    void* out;
    int64_t heads;
    int64_t si[4], so[4];  // element strides: batch, token, head, element
};

struct RotaryArgs {
    RotaryJob job[2];
    const int32_t* pos;
    const double* freq;
    int64_t pos_b, pos_t, freq_s;
    int64_t T, tokens;  // tokens = B * T
    int64_t groups;     // per token: turned groups, then copied groups
    int64_t turned;     // groups that are turned
    int64_t half;       // pairs = R / 2
    int64_t heads_per;  // heads of the combined list (q's, then k's) a block walks over
    int inverse;
};

// One head vector of the combined list: q's heads, then k's.
__device__ __forceinline__ int64_t head_in(RotaryArgs const& a, int64_t b, int64_t t, int64_t h, const void*& p) {
    bool const k = h >= a.job[0].heads;
    p = k ? a.job[1].in : a.job[0].in;
    int64_t const hh = k ? h - a.job[0].heads : h;
    return b * (k ? a.job[1].si[0] : a.job[0].si[0]) + t * (k ? a.job[1].si[1] : a.job[0].si[1]) +
           hh * (k ? a.job[1].si[2] : a.job[0].si[2]);
}
__device__ __forceinline__ int64_t head_out(RotaryArgs const& a, int64_t b, int64_t t, int64_t h, void*& p) {
    bool const k = h >= a.job[0].heads;
    p = k ? a.job[1].out : a.job[0].out;
    int64_t const hh = k ? h - a.job[0].heads : h;
    return b * (k ? a.job[1].so[0] : a.job[0].so[0]) + t * (k ? a.job[1].so[1] : a.job[0].so[1]) +
           hh * (k ? a.job[1].so[2] : a.job[0].so[2]);
}

__device__ __forceinline__ void angle_cs(double a, float& c, float& s) {
    double const turns = a * 0.15915494309189535, part = turns - rint(turns);  // 1 / (2 pi)
    // quarters of a turn are taken off in 64 bits, so that rounding costs 2^-28 turns and not 2^-26
    float const quarters = rintf(4.0f * static_cast<float>(part));
    float x, y;
    sincospif(static_cast<float>(2.0 * part - 0.5 * quarters), &y, &x);
    int const k = static_cast<int>(quarters) & 3;
    c = (k & 1) != 0 ? y : x;
    s = (k & 1) != 0 ? x : y;
    if (((k + 1) & 2) != 0) c = -c;
    if ((k & 2) != 0) s = -s;
}
__device__ __forceinline__ void angle_cs(double a, double& c, double& s) { sincos(a, &s, &c); }

// VP pairs a thread. VEC: unit strides and 16-byte vectors; interleaved pairs
// are 2*VP contiguous elements, halves VP contiguous elements in each half.
template <typename T, int VP, bool VEC, bool HALVES>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, T mag) {
    using V = typename Vec16<T>::type;
    constexpr int NV = Vec16<T>::n;
    constexpr int E = 2 * VP;
    prior_kernels_done();
    int64_t const id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (id >= a.tokens * a.groups) return;
    int64_t const token = id / a.groups, grp = id - token * a.groups;
    int64_t const b = token / a.T, t = token - b * a.T;
    bool const turn = grp < a.turned;

    // Element index of the group's first half (or its 2*VP elements) and of its second.
    int64_t e0, e1;
    if (turn) {
        e0 = HALVES ? grp * VP : grp * E;
        e1 = HALVES ? a.half + grp * VP : grp * E + VP;
    } else {
        e0 = 2 * a.half + (grp - a.turned) * E;
        e1 = e0 + VP;
    }
    T c[VP], s[VP];
    if (turn) {
        double const pos = static_cast<double>(a.pos[b * a.pos_b + t * a.pos_t]);
#pragma unroll
        for (int k = 0; k < VP; ++k) {
            angle_cs(pos * a.freq[(grp * VP + k) * a.freq_s], c[k], s[k]);
            c[k] *= mag;
            s[k] *= a.inverse ? -mag : mag;
        }
    }
    int64_t const heads = a.job[0].heads + a.job[1].heads;
    int64_t const h0 = static_cast<int64_t>(blockIdx.y) * a.heads_per;
    int64_t const h1 = min(heads, h0 + a.heads_per);
    for (int64_t h = h0; h < h1; h += kHeadsAtOnce) {
        T x[kHeadsAtOnce][E];
#pragma unroll
        for (int u = 0; u < kHeadsAtOnce; ++u) {
            if (h + u >= h1) break;
            const void* base;
            int64_t const off = head_in(a, b, t, h + u, base);
            T const* in = static_cast<T const*>(base) + off;
            if constexpr (VEC) {
#pragma unroll
                for (int v = 0; v < VP / NV; ++v) {
                    *reinterpret_cast<V*>(&x[u][v * NV]) = *reinterpret_cast<V const*>(in + e0 + v * NV);
                    *reinterpret_cast<V*>(&x[u][VP + v * NV]) = *reinterpret_cast<V const*>(in + e1 + v * NV);
                }
            } else {
                int64_t const step = h + u >= a.job[0].heads ? a.job[1].si[3] : a.job[0].si[3];
#pragma unroll
                for (int v = 0; v < VP; ++v) {
                    x[u][v] = in[(e0 + v) * step];
                    x[u][VP + v] = in[(e1 + v) * step];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kHeadsAtOnce; ++u) {
            if (h + u >= h1) break;
            if (turn) {
#pragma unroll
                for (int k = 0; k < VP; ++k) {
                    constexpr int step = HALVES ? 1 : 2, other = HALVES ? VP : 1;
                    T const x0 = x[u][step * k], x1 = x[u][step * k + other];
                    x[u][step * k] = x0 * c[k] - x1 * s[k];
                    x[u][step * k + other] = x0 * s[k] + x1 * c[k];
                }
            }
            void* base;
            int64_t const off = head_out(a, b, t, h + u, base);
            T* out = static_cast<T*>(base) + off;
            if constexpr (VEC) {
#pragma unroll
                for (int v = 0; v < VP / NV; ++v) {
                    *reinterpret_cast<V*>(out + e0 + v * NV) = *reinterpret_cast<V const*>(&x[u][v * NV]);
                    *reinterpret_cast<V*>(out + e1 + v * NV) = *reinterpret_cast<V const*>(&x[u][VP + v * NV]);
                }
            } else {
                int64_t const step = h + u >= a.job[0].heads ? a.job[1].so[3] : a.job[0].so[3];
#pragma unroll
                for (int v = 0; v < VP; ++v) {
                    out[(e0 + v) * step] = x[u][v];
                    out[(e1 + v) * step] = x[u][VP + v];
                }
            }
        }
    }
}

template <typename T>
bool rows_aligned(const RotaryJob& j) {
    if (j.heads == 0) return true;
    if (j.si[3] != 1 || j.so[3] != 1 || !aligned(j.in, 16) || !aligned(j.out, 16)) return false;
    for (int i = 0; i < 3; ++i)
        if ((j.si[i] * sizeof(T)) % 16 != 0 || (j.so[i] * sizeof(T)) % 16 != 0) return false;
    return true;
}

template <typename T>
int rotary(ann_stream stream, const ann_view* q_v, const ann_view* k_v, const ann_view* pos_v, const ann_view* freq_v,
           const ann_view* oq_v, const ann_view* ok_v, int pairs, int layout, T mag, int inverse) {
    Dims in[2], out[2], pos, freq;
    ANN_TRY(to_dims_flat(q_v, sizeof(T), "rotary q", in[0]));
    ANN_TRY(to_dims_flat(oq_v, sizeof(T), "rotary output q", out[0]));
    if ((k_v == nullptr) != (ok_v == nullptr)) return fail(ANN_EINVAL, "rotary: k and its output come together.");
    int const n = k_v != nullptr ? 2 : 1;
    if (n == 2) {
        ANN_TRY(to_dims_flat(k_v, sizeof(T), "rotary k", in[1]));
        ANN_TRY(to_dims_flat(ok_v, sizeof(T), "rotary output k", out[1]));
    }
    ANN_TRY(to_dims_flat(pos_v, sizeof(int32_t), "rotary positions", pos));
    ANN_TRY(to_dims_flat(freq_v, sizeof(double), "rotary frequencies", freq));
    if (pairs != ANN_ROTARY_INTERLEAVED && pairs != ANN_ROTARY_HALVES) return fail(ANN_EINVAL, "rotary pairs are invalid.");
    if (layout != ANN_LAYOUT_BTHD && layout != ANN_LAYOUT_BHTD) return fail(ANN_EINVAL, "rotary layout is invalid.");
    int const ta = layout == ANN_LAYOUT_BTHD ? 1 : 2, ha = 3 - ta;
    for (int k = 0; k < n; ++k) {
        if (in[k].rank != 4 || !same_extents(in[k], out[k]))
            return fail(ANN_EINVAL, "rotary expects rank-4 BTHD or BHTD tensors and outputs of the same extents.");
        if (!writable(out[k])) return fail(ANN_EINVAL, "rotary: an output axis has a zero pitch.");
        if (in[k].ext[0] != in[0].ext[0] || in[k].ext[ta] != in[0].ext[ta] || in[k].ext[3] != in[0].ext[3])
            return fail(ANN_EINVAL, "rotary: q %s and k %s differ in more than their heads.", extents_str(in[0]).c_str(),
                        extents_str(in[k]).c_str());
    }
    int64_t const B = in[0].ext[0], T_ = in[0].ext[ta], D = in[0].ext[3];
    bool const pos_ok = (pos.rank == 2 && pos.ext[0] == B && pos.ext[1] == T_) || (pos.rank == 1 && pos.ext[0] == T_);
    if (!pos_ok) return fail(ANN_EINVAL, "rotary positions must be [batch, tokens] or [tokens].");
    if (D % 2 != 0) return fail(ANN_EINVAL, "rotary requires an even head dimension.");
    if (freq.rank != 1 || 2 * freq.ext[0] > D)
        return fail(ANN_EINVAL, "rotary frequencies must be rank 1 with at most headDim/2 pairs.");

    RotaryArgs a{};
    for (int k = 0; k < n; ++k) {
        RotaryJob& j = a.job[k];
        j.in = in[k].data;
        j.out = out[k].data;
        j.heads = in[k].ext[ha];
        int const axis[4] = {0, ta, ha, 3};
        for (int i = 0; i < 4; ++i) {
            j.si[i] = in[k].str[axis[i]];
            j.so[i] = out[k].str[axis[i]];
        }
    }
    int64_t const heads = a.job[0].heads + a.job[1].heads;
    if (B == 0 || T_ == 0 || D == 0 || heads == 0) return ANN_OK;
    a.pos = static_cast<const int32_t*>(pos.data);
    a.pos_b = pos.rank == 2 ? pos.str[0] : 0;
    a.pos_t = pos.rank == 2 ? pos.str[1] : pos.str[0];
    a.freq = static_cast<const double*>(freq.data);
    a.freq_s = freq.str[0];
    a.T = T_;
    a.tokens = B * T_;
    a.half = freq.ext[0];
    a.inverse = inverse != 0;

    // A vector thread takes one 16-byte vector of each half: 2 NV elements. Both
    // the turned part and the rest have to be whole groups, the halves aligned.
    constexpr int NV = Vec16<T>::n;
    int64_t const rest = D - 2 * a.half;
    bool const vec = rows_aligned<T>(a.job[0]) && rows_aligned<T>(a.job[1]) && a.half % NV == 0 && rest % (2 * NV) == 0;
    int const vp = vec ? NV : 1;
    a.turned = a.half / vp;
    a.groups = a.turned + rest / (2 * vp);
    int64_t const threads = a.tokens * a.groups;
    // Heads a thread walks over: enough threads for four blocks of 256 an SM
    // first, then as many heads as possible, so that the angles are formed once
    // (at 4 x 4096 tokens and 64 heads: all heads of a token in one thread).
    int64_t const want = static_cast<int64_t>(sm_count()) * 4 * kThreads;
    int64_t per = ceil_div(heads * threads, want);
    per = std::min<int64_t>(heads, std::max<int64_t>(kHeadsAtOnce, ceil_div(per, kHeadsAtOnce) * kHeadsAtOnce));
    per = std::max(per, ceil_div(heads, 65535));
    a.heads_per = per;
    int64_t const gx = ceil_div(threads, kThreads);
    if (gx > INT32_MAX) return fail(ANN_ENOTSUP, "rotary: too many tokens for one call.");
    dim3 const grid(static_cast<unsigned>(gx), static_cast<unsigned>(ceil_div(heads, per)));
    if (threads > 0) {
        bool const halves = pairs == ANN_ROTARY_HALVES;
        auto const kernel = vec ? (halves ? rotary_kernel<T, NV, true, true> : rotary_kernel<T, NV, true, false>)
                                : (halves ? rotary_kernel<T, 1, false, true> : rotary_kernel<T, 1, false, false>);
        launch_overlapping(kernel, grid, kThreads, 0, as_stream(stream), a, mag);
    }
    return check_launch("rotary");
}

__global__ void frequencies_kernel(double* f, int64_t stride, int64_t n, double base, double factor, double trained,
                                   double low, double high) {
    int64_t const p = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (p >= n) return;
    double v = pow(base, -static_cast<double>(p) / static_cast<double>(n));
    if (trained > 0.0) {
        double const turns = trained * v * 0.15915494309189535;  // full turns over the trained length
        double const w = fmin(fmax((turns - low) / (high - low), 0.0), 1.0);
        v *= w + (1.0 - w) / factor;
    } else {
        v /= factor;
    }
    f[p * stride] = v;
}

int frequencies(ann_stream stream, const ann_view* f_v, double base, double factor, double trained, double low,
                double high) {
    Dims f;
    ANN_TRY(to_dims_flat(f_v, sizeof(double), "rotaryFrequencies", f));
    if (f.rank != 1) return fail(ANN_EINVAL, "rotaryFrequencies expects a rank-1 output.");
    if (!writable(f)) return fail(ANN_EINVAL, "rotaryFrequencies: the output has a zero pitch.");
    if (!(base > 0.0) || !std::isfinite(base) || !(factor > 0.0) || !std::isfinite(factor))
        return fail(ANN_EINVAL, "rotaryFrequencies: base and factor must be positive and finite.");
    if (!(trained >= 0.0) || !std::isfinite(trained))
        return fail(ANN_EINVAL, "rotaryFrequencies: the trained length must not be negative.");
    if (trained > 0.0 && !(low < high && std::isfinite(low) && std::isfinite(high)))
        return fail(ANN_EINVAL, "rotaryFrequencies needs lowTurns < highTurns.");
    int64_t const n = f.ext[0];
    if (n == 0) return ANN_OK;
    frequencies_kernel<<<static_cast<unsigned>(ceil_div(n, 128)), 128, 0, as_stream(stream)>>>(
        static_cast<double*>(f.data), f.str[0], n, base, factor, trained, low, high);
    return check_launch("rotaryFrequencies");
}

}  // namespace
}  // namespace ann

extern "C" {

int ann_rotary_f32(ann_stream s, const ann_view* q, const ann_view* k, const ann_view* positions,
                   const ann_view* frequencies, const ann_view* out_q, const ann_view* out_k, int32_t pairs,
                   int32_t layout, float magnitude, int32_t inverse) {
    ANN_API_BEGIN
    return ann::rotary<float>(s, q, k, positions, frequencies, out_q, out_k, pairs, layout, magnitude, inverse);
    ANN_API_END
}
int ann_rotary_f64(ann_stream s, const ann_view* q, const ann_view* k, const ann_view* positions,
                   const ann_view* frequencies, const ann_view* out_q, const ann_view* out_k, int32_t pairs,
                   int32_t layout, double magnitude, int32_t inverse) {
    ANN_API_BEGIN
    return ann::rotary<double>(s, q, k, positions, frequencies, out_q, out_k, pairs, layout, magnitude, inverse);
    ANN_API_END
}
int ann_rotary_frequencies(ann_stream s, const ann_view* frequencies, double base, double factor,
                           double trained_length, double low_turns, double high_turns) {
    ANN_API_BEGIN
    return ann::frequencies(s, frequencies, base, factor, trained_length, low_turns, high_turns);
    ANN_API_END
}

}  // extern "C"
