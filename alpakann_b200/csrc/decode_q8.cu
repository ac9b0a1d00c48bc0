// decode_q8.cu -- attention of the last tokens over a KV cache held in 8 bits.
//
// Query i of Tq (the last tokens of a sequence of `length` keys) and head hq:
//   s_j = scale * ks[j / block] * (q . n_j),  j < length - Tq + 1 + i  (causal) or j < length
//   out = sum_j e^(s_j - max s) vs[j / block] m_j / sum_j e^(s_j - max s)
// with n_j, m_j the cache's whole numbers (kv_q8.cu). A query that sees no key
// gets a row of zeros.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <set>

#include "common.cuh"
#include "reduce.cuh"

namespace cg = cooperative_groups;

namespace ann {
namespace {

struct DecodeQ8Args {
    const float* q;
    const int8_t* k;
    const int8_t* v;
    const float* ks;
    const float* vs;
    float* out;
    const int32_t* lengths;  // may be null: the whole cache
    int64_t len_s;
    int64_t q_b, q_t, q_h;       // element strides (unit stride along d)
    int64_t o_b, o_t, o_h, o_d;
    int64_t k_b, k_h, k_t;
    int64_t v_b, v_h, v_t;
    int64_t ks_b, ks_h, ks_j;
    int64_t vs_b, vs_h, vs_j;
    int64_t B, Tq, Hq, Hkv, cap;
    uint32_t g;
    int64_t row_tiles;  // CTAs for the Tq * g rows of a KV head
    int splits;         // of the key range
    int block_shift, causal;
    float scale;
};

// How the products are formed. An int8 value is exact in fp16, a float32 value is
// the sum of two fp16 parts (11 bits each, the row scaled by a power of two so
// that both are normal numbers), and mma.sync adds exact products of fp16 in
// float32. An m16n8k16 product takes 16 rows: eight query rows' high parts and
// the same rows' low parts, so one instruction gives both halves of eight rows,
// in the same thread, at float32 accuracy. The probabilities go through the same
// split on their way to the product with V.
//
// How the cache reaches the fragments. The order of the summed index and of the
// output columns of a matrix product is free as long as both operands agree, so
// a lane takes the bytes that one wide load gives it: 16 consecutive elements of
// a key's row for q.k (four lanes cover 64 bytes of a key), 16 consecutive
// elements of four keys for p.v (eight lanes cover a row). No shared memory, no
// transposition: a warp loads its keys straight to registers, the next tile's
// while it works on this one.
//
// Every warp takes tiles of KT keys of its own, keeps a running maximum and sum
// per row (base 2), and adds each tile's p.v from a fresh accumulator, so no sum
// of more than KT products is left to the tensor core's own rounding. Warps meet
// in shared memory, the CTAs of a cluster (the key range's splits) in
// distributed shared memory; no scratch memory, no atomics, one launch, and a
// fixed order of sums.
constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int MT>
struct Q8 {
    static constexpr int KT = D <= 128 ? 32 : 16;  // keys per tile of a warp
    static constexpr int ROWS = 8 * MT;            // query rows of a CTA
    static constexpr int KS = D / 16;              // k16 steps of q.k
    static constexpr int NK = KT / 8;              // n8 tiles of keys
    static constexpr int KV = KT / 16;             // k16 steps of p.v, groups of 16 keys
    static constexpr int VW = D / 32;              // words of V per lane and key
    static constexpr int KW = D / 16;              // words of K per lane and key
    static constexpr bool QREG = MT * KS <= 8;     // q's fragments in registers
    static constexpr size_t OFF_Q = 0;                                        // uint4 [MT][KS][32]
    static constexpr size_t OFF_O = OFF_Q + size_t{16} * MT * KS * 32;        // float [kWarps][ROWS][D]
    static constexpr size_t OFF_ML = OFF_O + sizeof(float) * kWarps * ROWS * D;  // float [2][kWarps][ROWS]
    static constexpr size_t OFF_F = OFF_ML + sizeof(float) * 2 * kWarps * ROWS;  // float [ROWS]: score factors
    static constexpr size_t OFF_X = OFF_F + sizeof(float) * ROWS;             // float [2][ROWS]: this CTA's max, sum
    static constexpr size_t OFF_W = OFF_X + sizeof(float) * 2 * ROWS;         // float [kMaxCluster][ROWS], then [ROWS]
    static constexpr size_t SMEM = OFF_W + sizeof(float) * (kMaxCluster + 1) * ROWS;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two unsigned bytes u (= n + 128) of w picked by `sel` as fp16 whole numbers n:
// 0x6400 | u is 1024 + u, and 1024 + 128 is taken off, all exact.
__device__ __forceinline__ uint32_t halves_of(uint32_t w, uint32_t sel) {
    uint32_t const biased = __byte_perm(w, 0x64646464u, sel);
    __half2 const h = __hsub2(*reinterpret_cast<__half2 const*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<uint32_t const*>(&h);
}

// x, y -> their fp16 parts, high and low, each as a pair.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    __half2 const h = __floats2half2_rn(x, y);
    float2 const f = __half22float2(h);
    __half2 const l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<uint32_t const*>(&h);
    lo = *reinterpret_cast<uint32_t const*>(&l);
}

__device__ __forceinline__ uint4 load16(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 load8(const int8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// 2^(e - 127) for a biased exponent e in [1, 254].
__device__ __forceinline__ float pow2_biased(int e) { return __int_as_float(e << 23); }

template <int D, int MT>
__global__ void __launch_bounds__(kThreads, MT == 1 && D <= 128 ? 3 : 2) decode_q8_kernel(DecodeQ8Args a) {
    using C = Q8<D, MT>;
    extern __shared__ __align__(16) unsigned char smem[];
    uint4* sq = reinterpret_cast<uint4*>(smem + C::OFF_Q);
    float* so = reinterpret_cast<float*>(smem + C::OFF_O);
    float* sml = reinterpret_cast<float*>(smem + C::OFF_ML);
    float* sf = reinterpret_cast<float*>(smem + C::OFF_F);
    float* sx = reinterpret_cast<float*>(smem + C::OFF_X);
    float* sw = reinterpret_cast<float*>(smem + C::OFF_W);
    int const tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int const split = static_cast<int>(blockIdx.x) % a.splits;
    int64_t unit = blockIdx.x / a.splits;
    int64_t const row0 = (unit % a.row_tiles) * C::ROWS;  // first of the KV head's Tq * g query rows
    unit /= a.row_tiles;
    int64_t const kvh = unit % a.Hkv, b = unit / a.Hkv;
    int64_t const left = a.Tq * a.g - row0;
    int const rows = static_cast<int>(min(left, int64_t{C::ROWS}));

    int64_t len = a.cap;
    if (a.lengths != nullptr) len = min(a.cap, max(int64_t{0}, static_cast<int64_t>(a.lengths[b * a.len_s])));
    // keys that row r of the tile sees; rows are ordered by token, then head
    auto visible = [&](int r) {
        int64_t const n = a.causal ? len - a.Tq + 1 + (row0 + r) / a.g : len;
        return static_cast<int>(max(int64_t{0}, n));
    };
    int const most = visible(rows - 1), least = visible(0);

    // q's fragments and the factor of each row's scores.
    for (int r = warp; r < C::ROWS; r += kWarps) {
        int64_t const row = row0 + r, hq = kvh * a.g + row % a.g;
        bool const given = r < rows && hq < a.Hq;
        float const* q = a.q + b * a.q_b + (row / a.g) * a.q_t + hq * a.q_h;
        float4 x[(D + 127) / 128];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < (D + 127) / 128; ++i) {
            int const d = 128 * i + 4 * lane;
            x[i] = given && d < D ? *reinterpret_cast<float4 const*>(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
        }
        top = warp_max(top);
        // largest value into [2^13, 2^14): e = its biased exponent, held where the factors stay normal
        int e = static_cast<int>(__float_as_uint(top) >> 23);
        e = e == 255 ? 140 : max(e, 15);
        float const up = pow2_biased(267 - e), down = pow2_biased(e - 13);  // 2^(140 - e), 2^(e - 140)
        if (lane == 0) sf[r] = down * (a.scale * kLog2e);
#pragma unroll
        for (int i = 0; i < (D + 127) / 128; ++i) {
            int const d = 128 * i + 4 * lane;
            if (d >= D) continue;
            uint4 f;
            split2(x[i].x * up, x[i].y * up, f.x, f.y);
            split2(x[i].z * up, x[i].w * up, f.z, f.w);
            // element d = 64 c + 16 t' + 4 w of row g' sits in step 4 c + w, lane (g', t')
            int const step = (d / 64) * 4 + (d / 4) % 4, to = (r & 7) * 4 + (d / 16) % 4;
            sq[((r >> 3) * C::KS + step) * 32 + to] = f;
        }
    }
    __syncthreads();
    uint4 qf[C::QREG ? MT * C::KS : 1];
    if constexpr (C::QREG) {
#pragma unroll
        for (int i = 0; i < MT * C::KS; ++i) qf[i] = sq[i * 32 + lane];
    }
    float fac[MT];
    int seen[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        fac[m] = sf[8 * m + g];
        seen[m] = 8 * m + g < rows ? visible(8 * m + g) : 0;
    }

    int8_t const* kb = a.k + b * a.k_b + kvh * a.k_h;
    int8_t const* vb = a.v + b * a.v_b + kvh * a.v_h;
    float const* ks = a.ks + b * a.ks_b + kvh * a.ks_h;
    float const* vs = a.vs + b * a.vs_b + kvh * a.vs_h;

    int const tiles = (most + C::KT - 1) / C::KT;
    int const t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
    int const t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);

    uint32_t kr[C::NK][C::KW], vr[C::KV][4][C::VW];
    float ksc[C::KV], vsc[C::KV];
    auto load_k = [&](int tile) {
#pragma unroll
        for (int j = 0; j < C::NK; ++j) {
            int64_t const key = min(tile * C::KT + 8 * j + g, most - 1);  // masked keys read the last seen one
            int8_t const* p = kb + key * a.k_t + 16 * t;
#pragma unroll
            for (int i = 0; i < C::KW / 4; ++i) {
                uint4 const w = load16(p + 64 * i);
                kr[j][4 * i] = w.x, kr[j][4 * i + 1] = w.y, kr[j][4 * i + 2] = w.z, kr[j][4 * i + 3] = w.w;
            }
        }
#pragma unroll
        for (int i = 0; i < C::KV; ++i)
            ksc[i] = ks[static_cast<int64_t>(min(tile * C::KT + 16 * i, most - 1) >> a.block_shift) * a.ks_j];
    };
    auto load_v = [&](int tile) {
#pragma unroll
        for (int i = 0; i < C::KV; ++i) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                int64_t const key = min(tile * C::KT + 16 * i + 2 * t + (x & 1) + 8 * (x >> 1), most - 1);
                if constexpr (D == 64) {
                    uint2 const w = load8(vb + key * a.v_t + 8 * g);
                    vr[i][x][0] = w.x, vr[i][x][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < C::VW / 4; ++c) {
                        uint4 const w = load16(vb + key * a.v_t + 128 * c + 16 * g);
                        vr[i][x][4 * c] = w.x, vr[i][x][4 * c + 1] = w.y;
                        vr[i][x][4 * c + 2] = w.z, vr[i][x][4 * c + 3] = w.w;
                    }
                }
            }
            vsc[i] = vs[static_cast<int64_t>(min(tile * C::KT + 16 * i, most - 1) >> a.block_shift) * a.vs_j];
        }
    };

    float m_run[MT], l_run[MT], o[MT][D / 8][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        m_run[m] = neg_inf(0.0f);
        l_run[m] = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[m][n][0] = o[m][n][1] = 0.0f;
    }

    int tile = t0 + warp;
    if (tile < t1) {
        load_k(tile);
        load_v(tile);
    }
    for (; tile < t1; tile += kWarps) {
        bool const more = tile + kWarps < t1;
        // scores of 8 MT rows and KT keys
        float s[MT][C::NK][2];
#pragma unroll
        for (int j = 0; j < C::NK; ++j) {
            float c[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0.0f;
#pragma unroll
            for (int st = 0; st < C::KS; ++st) {
                uint32_t const w = kr[j][st] ^ 0x80808080u;
                uint32_t const b0 = halves_of(w, 0x4140), b1 = halves_of(w, 0x4342);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    uint4 const q = C::QREG ? qf[m * C::KS + st] : sq[(m * C::KS + st) * 32 + lane];
                    mma16816(c[m], q.x, q.y, q.z, q.w, b0, b1);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float const f = fac[m] * ksc[j / 2];
                s[m][j][0] = (c[m][0] + c[m][2]) * f;
                s[m][j][1] = (c[m][1] + c[m][3]) * f;
            }
        }
        if (more) load_k(tile + kWarps);
        if ((tile + 1) * C::KT > least) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < C::NK; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (tile * C::KT + 8 * j + 2 * t + e >= seen[m]) s[m][j][e] = neg_inf(0.0f);
        }
        // V's scales relative to a power of two, so that p * scale fits fp16
        float vtop = 0.0f;
#pragma unroll
        for (int i = 0; i < C::KV; ++i) vtop = fmaxf(vtop, fabsf(vsc[i]));
        int const ve = min(max(static_cast<int>(__float_as_uint(vtop) >> 23), 15), 253);
        float const vdown = pow2_biased(254 - ve), back = pow2_biased(ve - 13);
        uint32_t pa[MT][C::KV][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float top = neg_inf(0.0f);
#pragma unroll
            for (int j = 0; j < C::NK; ++j) top = fmaxf(top, fmaxf(s[m][j][0], s[m][j][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float const m_new = fmaxf(m_run[m], top);
            float const base = m_new == neg_inf(0.0f) ? 0.0f : m_new;
            if (__any_sync(0xffffffffu, m_new > m_run[m])) {
                float const alpha = exp2f(m_run[m] - base);
                l_run[m] *= alpha;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) o[m][n][0] *= alpha, o[m][n][1] *= alpha;
                m_run[m] = m_new;
            }
#pragma unroll
            for (int i = 0; i < C::KV; ++i) {
                float const w = vsc[i] * vdown * 8192.0f;  // p * w < 2^14
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float const p0 = exp2f(s[m][2 * i + h][0] - base), p1 = exp2f(s[m][2 * i + h][1] - base);
                    l_run[m] += p0 + p1;
                    split2(p0 * w, p1 * w, pa[m][i][2 * h], pa[m][i][2 * h + 1]);
                }
            }
        }
        // o += p V, one word of V (four columns of lanes) at a time
#pragma unroll
        for (int w = 0; w < C::VW; ++w) {
            float c[MT][4][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n) c[m][n][0] = c[m][n][1] = c[m][n][2] = c[m][n][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < C::KV; ++i) {
                uint32_t const v0 = vr[i][0][w] ^ 0x80808080u, v1 = vr[i][1][w] ^ 0x80808080u;
                uint32_t const v2 = vr[i][2][w] ^ 0x80808080u, v3 = vr[i][3][w] ^ 0x80808080u;
                uint32_t const x01 = __byte_perm(v0, v1, 0x5140), y01 = __byte_perm(v0, v1, 0x7362);
                uint32_t const x23 = __byte_perm(v2, v3, 0x5140), y23 = __byte_perm(v2, v3, 0x7362);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint32_t const b0 = halves_of(n < 2 ? x01 : y01, n % 2 ? 0x4342 : 0x4140);
                    uint32_t const b1 = halves_of(n < 2 ? x23 : y23, n % 2 ? 0x4342 : 0x4140);
#pragma unroll
                    for (int m = 0; m < MT; ++m)
                        mma16816(c[m][n], pa[m][i][0], pa[m][i][1], pa[m][i][2], pa[m][i][3], b0, b1);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    o[m][4 * w + n][0] = fmaf(c[m][n][0] + c[m][n][2], back, o[m][4 * w + n][0]);
                    o[m][4 * w + n][1] = fmaf(c[m][n][1] + c[m][n][3], back, o[m][4 * w + n][1]);
                }
        }
        if (more) load_v(tile + kWarps);
    }

    // Warps to CTA: every warp's rows, maxima and sums in shared memory.
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float l = l_run[m];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            sml[warp * C::ROWS + 8 * m + g] = m_run[m];
            sml[(kWarps + warp) * C::ROWS + 8 * m + g] = l;
        }
        // columns 2t and 2t + 1 of n-tile n are elements 32 t + n and 32 t + 16 + n of a
        // 128-element stretch (D = 64: 16 t + n and 16 t + 8 + n)
        float* row = so + (warp * C::ROWS + 8 * m + g) * D;
        constexpr int STRETCH = D == 64 ? 8 : 16;
#pragma unroll
        for (int n = 0; n < D / 8; n += 4) {
            float* p = row + (n / STRETCH) * 128 + 2 * STRETCH * t + n % STRETCH;
            *reinterpret_cast<float4*>(p) = make_float4(o[m][n][0], o[m][n + 1][0], o[m][n + 2][0], o[m][n + 3][0]);
            *reinterpret_cast<float4*>(p + STRETCH) =
                make_float4(o[m][n][1], o[m][n + 1][1], o[m][n + 2][1], o[m][n + 3][1]);
        }
    }
    __syncthreads();
    auto weight = [](float m, float top) { return top == neg_inf(0.0f) ? 0.0f : exp2f(m - top); };
    if (tid < C::ROWS) {
        float top = neg_inf(0.0f), l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sml[w * C::ROWS + tid]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            float const f = weight(sml[w * C::ROWS + tid], top);
            l += f * sml[(kWarps + w) * C::ROWS + tid];
            sml[w * C::ROWS + tid] = f;
        }
        sx[tid] = top;
        sx[C::ROWS + tid] = l;
    }
    __syncthreads();
    auto sum_warps = [&](int i) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) v = fmaf(sml[w * C::ROWS + i / D], so[w * C::ROWS * D + i], v);
        return v;
    };
    auto store = [&](int i, float v) {
        int const r = i / D, d = i - r * D;
        int64_t const row = row0 + r, hq = kvh * a.g + row % a.g;
        if (hq < a.Hq) a.out[b * a.o_b + (row / a.g) * a.o_t + hq * a.o_h + d * a.o_d] = v;
    };
    if (a.splits == 1) {
        for (int i = tid; i < rows * D; i += kThreads) {
            float const l = sx[C::ROWS + i / D];
            store(i, l == 0.0f ? 0.0f : sum_warps(i) / l);
        }
        return;
    }
    for (int i = tid; i < rows * D; i += kThreads) so[i] = sum_warps(i);

    // CTAs of the cluster: each gives its share of the rows' elements.
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (tid < rows) {
        float top = neg_inf(0.0f), l = 0.0f;
        for (int r = 0; r < a.splits; ++r) top = fmaxf(top, cluster.map_shared_rank(sx, r)[tid]);
        for (int r = 0; r < a.splits; ++r) {
            float const* px = cluster.map_shared_rank(sx, r);
            float const f = weight(px[tid], top);
            l += f * px[C::ROWS + tid];
            sw[r * C::ROWS + tid] = f;
        }
        sw[kMaxCluster * C::ROWS + tid] = l;
    }
    __syncthreads();
    int const lo = rows * D * split / a.splits, hi = rows * D * (split + 1) / a.splits;
    for (int i = lo + tid; i < hi; i += kThreads) {
        float v = 0.0f;
        for (int r = 0; r < a.splits; ++r) v = fmaf(sw[r * C::ROWS + i / D], cluster.map_shared_rank(so, r)[i], v);
        float const l = sw[kMaxCluster * C::ROWS + i / D];
        store(i, l == 0.0f ? 0.0f : v / l);
    }
    cluster.sync();  // peers' shared memory must outlive the reads above
}

// Splits of the key range = cluster size: enough CTAs for two on every SM, as
// long as a split keeps two tiles for each of its warps.
int choose_splits(int64_t units, int64_t cap, int tile) {
    int64_t const most = std::max<int64_t>(1, ceil_div(cap, int64_t{2} * tile * kWarps));
    int64_t const want = ceil_div(int64_t{2} * sm_count(), units);
    return static_cast<int>(std::min({most, want, int64_t{kMaxCluster}}));
}

template <int D, int MT>
int launch(ann_stream stream, DecodeQ8Args& a) {
    using C = Q8<D, MT>;
    static std::mutex mu;
    static std::set<int> ready;  // devices whose kernel attributes are set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8: no CUDA device.");
    {
        std::lock_guard<std::mutex> lock(mu);
        if (ready.count(dev) == 0) {
            cudaError_t e = cudaFuncSetAttribute(decode_q8_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(C::SMEM));
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(decode_q8_kernel<D, MT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8 setup: %s", cudaGetErrorString(e));
            ready.insert(dev);
        }
    }
    a.row_tiles = ceil_div(a.Tq * a.g, C::ROWS);
    int64_t const units = a.B * a.Hkv * a.row_tiles;
    a.splits = choose_splits(units, a.cap, C::KT);
    int64_t const grid = units * a.splits;
    if (grid > INT32_MAX) return fail(ANN_ENOTSUP, "attentionDecodeQ8: grid too large.");
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = as_stream(stream);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    cudaError_t const e = cudaLaunchKernelEx(&cfg, decode_q8_kernel<D, MT>, a);
    if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8: %s", cudaGetErrorString(e));
    return check_launch("attentionDecodeQ8");
}

template <int D>
int launch_rows(ann_stream stream, DecodeQ8Args& a) {
    return a.Tq * a.g <= 8 ? launch<D, 1>(stream, a) : launch<D, 2>(stream, a);
}

int decode_q8(ann_stream stream, const ann_view* q_v, const ann_view* k_v, const ann_view* v_v, const ann_view* ks_v,
              const ann_view* vs_v, const ann_view* len_v, const ann_view* o_v, float scale, uint32_t g, uint32_t block,
              int layout, int causal) {
    if (g == 0u) return fail(ANN_EINVAL, "attentionDecodeQ8 requires queriesPerKvGroup > 0.");
    if (layout != ANN_LAYOUT_BTHD && layout != ANN_LAYOUT_BHTD)
        return fail(ANN_EINVAL, "attentionDecodeQ8: invalid kv layout.");
    if (block == 0u) return fail(ANN_EINVAL, "attentionDecodeQ8 requires tokensPerScale > 0.");
    Dims q, k, v, ks, vs, o;
    ANN_TRY(to_dims(q_v, sizeof(float), "attentionDecodeQ8 Q", q));
    ANN_TRY(to_dims(k_v, 1, "attentionDecodeQ8 K", k));
    ANN_TRY(to_dims(v_v, 1, "attentionDecodeQ8 V", v));
    ANN_TRY(to_dims(ks_v, sizeof(float), "attentionDecodeQ8 K scales", ks));
    ANN_TRY(to_dims(vs_v, sizeof(float), "attentionDecodeQ8 V scales", vs));
    ANN_TRY(to_dims(o_v, sizeof(float), "attentionDecodeQ8 out", o));
    if (q.rank != 4 || k.rank != 4 || v.rank != 4 || o.rank != 4 || ks.rank != 3 || vs.rank != 3)
        return fail(ANN_EINVAL, "attentionDecodeQ8 expects rank-4 tensors and rank-3 scales.");
    if (!same_extents(q, o)) return fail(ANN_EINVAL, "attentionDecodeQ8: out must have the extents of Q.");
    if (!writable(o)) return fail(ANN_EINVAL, "attentionDecodeQ8: an axis of out has a zero pitch.");
    if (!same_extents(k, v)) return fail(ANN_EINVAL, "attentionDecodeQ8: K and V extents differ.");
    int const tok = layout == ANN_LAYOUT_BTHD ? 1 : 2, head = 3 - tok;
    int64_t const B = q.ext[0], Hq = q.ext[2], D = q.ext[3];
    if (k.ext[0] != B || k.ext[3] != D || k.ext[head] <= (Hq - 1) / static_cast<int64_t>(g))
        return fail(ANN_EINVAL, "attentionDecodeQ8: Q %s does not match K/V %s.", extents_str(q).c_str(),
                    extents_str(k).c_str());
    for (const Dims* s : {&ks, &vs})
        if (s->ext[0] != B || s->ext[1] != k.ext[head] || s->ext[2] != ceil_div(k.ext[tok], block))
            return fail(ANN_EINVAL, "attentionDecodeQ8: scales %s do not match the cache %s with %u tokens a scale.",
                        extents_str(*s).c_str(), extents_str(k).c_str(), block);
    DecodeQ8Args a{};
    if (len_v != nullptr) {
        Dims len;
        ANN_TRY(to_dims(len_v, sizeof(int32_t), "attentionDecodeQ8 lengths", len));
        if (len.rank != 1 || len.ext[0] != B)
            return fail(ANN_EINVAL, "attentionDecodeQ8 lengths must be rank 1 with one entry per sequence.");
        a.lengths = static_cast<const int32_t*>(len.data);
        a.len_s = len.str[0];
    }
    if (q.numel() == 0) return ANN_OK;
    if (D != 64 && D != 128 && D != 256)
        return fail(ANN_ENOTSUP, "attentionDecodeQ8: head dim %lld not supported.", static_cast<long long>(D));
    if (block < 16 || (block & (block - 1)) != 0)
        return fail(ANN_ENOTSUP, "attentionDecodeQ8 needs tokensPerScale to be a power of two of 16 or more.");
    if (q.str[3] != 1 || k.str[3] != 1 || v.str[3] != 1 || !aligned(q.data, 16) || !aligned(k.data, 16) ||
        !aligned(v.data, 16))
        return fail(ANN_ENOTSUP, "attentionDecodeQ8 needs unit-stride head vectors and 16-byte aligned rows.");
    for (int i = 0; i < 3; ++i)
        if (q.str[i] % 4 != 0 || k.str[i] % 16 != 0 || v.str[i] % 16 != 0)
            return fail(ANN_ENOTSUP, "attentionDecodeQ8 needs unit-stride head vectors and 16-byte aligned rows.");
    a.q = static_cast<const float*>(q.data);
    a.k = static_cast<const int8_t*>(k.data);
    a.v = static_cast<const int8_t*>(v.data);
    a.ks = static_cast<const float*>(ks.data);
    a.vs = static_cast<const float*>(vs.data);
    a.out = static_cast<float*>(o.data);
    a.q_b = q.str[0], a.q_t = q.str[1], a.q_h = q.str[2];
    a.o_b = o.str[0], a.o_t = o.str[1], a.o_h = o.str[2], a.o_d = o.str[3];
    a.k_b = k.str[0], a.k_h = k.str[head], a.k_t = k.str[tok];
    a.v_b = v.str[0], a.v_h = v.str[head], a.v_t = v.str[tok];
    a.ks_b = ks.str[0], a.ks_h = ks.str[1], a.ks_j = ks.str[2];
    a.vs_b = vs.str[0], a.vs_h = vs.str[1], a.vs_j = vs.str[2];
    if (k.ext[tok] > (int64_t{1} << 30)) return fail(ANN_ENOTSUP, "attentionDecodeQ8: more than 2^30 keys.");
    a.B = B;
    a.Tq = q.ext[1];
    a.Hq = Hq;
    a.Hkv = ceil_div(Hq, static_cast<int64_t>(g));  // KV heads that queries read
    a.cap = k.ext[tok];
    a.g = g;
    a.block_shift = __builtin_ctz(block);
    a.causal = causal != 0;
    a.scale = scale;
    if (D == 64) return launch_rows<64>(stream, a);
    if (D == 128) return launch_rows<128>(stream, a);
    return launch_rows<256>(stream, a);
}

}  // namespace
}  // namespace ann

extern "C" {

int ann_attention_decode_q8_f32(ann_stream s, const ann_view* q, const ann_view* k_cache, const ann_view* v_cache,
                                const ann_view* k_scale, const ann_view* v_scale, const ann_view* lengths,
                                const ann_view* out, float scale, uint32_t queries_per_kv_group,
                                uint32_t tokens_per_scale, int32_t kv_layout, int32_t causal) {
    ANN_API_BEGIN
    return ann::decode_q8(s, q, k_cache, v_cache, k_scale, v_scale, lengths, out, scale, queries_per_kv_group,
                          tokens_per_scale, kv_layout, causal);
    ANN_API_END
}

}  // extern "C"
