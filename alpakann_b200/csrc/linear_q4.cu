// linear_q4.cu -- products with weights held in 4 bits.
//
// A weight W[k, n] (row-major [in, out], as linear's) is (u - 8) * s: u is its
// nibble, s the fp32 scale of its group of `group` consecutive inputs and its
// column. Eight consecutive inputs of a column share one 32-bit word, the first
// in the low bits:
//   packed [K / 8, N] int32, scales [ceil(K / group), N].
//   y[m, n] = act(sum_k x[m, k] W[k, n] + bias[n]) + residual[m, n]
#include <cooperative_groups.h>

#include <algorithm>
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

// The product in whole numbers. A nibble u is an 8-bit operand as it is: two
// masks unpack the eight of a word. A row of x is rounded to 31 bits of its
// largest value (over a warp's inputs) and cut into four 8-bit digits, and
// mma.sync.m16n8k32 on int8 multiplies, transposed: 16 columns of W by 8 slots,
// the slots being the digits of two rows. The sums are exact in int32, the offset
// of 8 included: a product with ones gives the digits' sums, of which eight times
// are taken off. They become fp32 when their group of inputs ends and meet its
// scale. The order of the summed index is free, so a lane takes the words as a
// 16-byte load gives them, eight inputs (its octet of 32) of four neighbouring
// columns; x's digits are laid out to match.
//
// A CTA stays and takes one tile of 32 CT columns after another. Each of its warps
// (and each CTA of a cluster, where columns are few) has inputs of its own, whose
// digits it prepares once; it streams their weights, 128 inputs at a time (a quad
// of products' depth), through a ring in shared memory (cp.async, on across tiles),
// 4 to 8 KB in flight a warp. The warps' sums of a
// tile meet in shared memory, across a cluster in the CTA that owns a share of the
// columns, which applies bias, activation and residual. One launch, no scratch
// memory, no atomics, a fixed order of sums.
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 16;
// Bytes of x's digits in a CTA: at most 68 steps of 32 inputs a warp, whose digits'
// products with nibbles, |u d| <= 1920, sum up to less than 2^23: 256 times that
// fits 32 bits.
constexpr size_t kMaxDigits = 136 << 10;

// Shared memory: rings [kWarps][DEPTH quads][4][CT][32] uint4, two buffers of sums
// [kWarps][ROWS][COLS] and of the cluster's [per * splits]; then per quad of the
// CTA digits uint2 [4][NT][32] and offsets int [4][NT][4].
template <int CT, int NT>
struct Q4 {
    static constexpr int COLS = 32 * CT, ROWS = 2 * NT, ITEMS = ROWS * COLS;
    static constexpr int DEPTH = 4 / CT;                            // quads in flight a warp
    static constexpr size_t RING = size_t{16} * DEPTH * 4 * CT * 32;  // of a warp
    static constexpr size_t OFF_S = RING * kWarps;
    static constexpr size_t OFF_R = OFF_S + sizeof(float) * 2 * kWarps * ITEMS;
    static constexpr size_t OFF_D = OFF_R + sizeof(float) * 2 * (ITEMS + kMaxCluster);
    static constexpr size_t ROOM = kMaxDigits < 227 * 1024 - OFF_D ? kMaxDigits : 227 * 1024 - OFF_D;
    static constexpr size_t QUAD = size_t{4} * NT * (32 * sizeof(uint2) + 4 * sizeof(int));
    // Quads of inputs whose digits fit the largest cluster's CTAs (a CTA's share may be one longer).
    static constexpr int64_t MAX_QUADS = kMaxCluster * (static_cast<int64_t>(ROOM / QUAD) - 1);
};

// c += a b, int8 products of depth 32, exact in int32.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// CT: 16-byte words of columns per lane (32 CT columns a tile); NT: slots / 8 (2 NT
// rows a CTA); VEC: words and scales of four columns are one aligned load.
template <int CT, int NT, bool VEC>
__global__ void __launch_bounds__(kThreads, NT * CT >= 4 ? 1 : 2) linear_q4_kernel(LinearQ4Args a) {
    using C = Q4<CT, NT>;
    extern __shared__ __align__(16) unsigned char smem[];
    int const tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int const split = static_cast<int>(blockIdx.x) % a.splits;
    if (a.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // "this CTA runs"
    int64_t const row0 = static_cast<int64_t>(blockIdx.y) * C::ROWS;
    // this warp's quads of 128 inputs, in steps of 32
    int const quads = static_cast<int>((a.K + 127) / 128), parts = a.splits * kWarps, part = split * kWarps + warp;
    int const first = static_cast<int>(static_cast<int64_t>(quads) * (split * kWarps) / parts);  // the CTA's first
    int const q0 = static_cast<int>(static_cast<int64_t>(quads) * part / parts);
    int const q1 = static_cast<int>(static_cast<int64_t>(quads) * (part + 1) / parts);
    int const s0 = 4 * q0, s1 = min(4 * q1, static_cast<int>((a.K + 31) / 32));
    int const octets = static_cast<int>(a.K / 8), per_group = a.group / 32;
    int const tiles = static_cast<int>((a.N + C::COLS - 1) / C::COLS);
    int const tile0 = static_cast<int>(blockIdx.x) / a.splits, stride = static_cast<int>(gridDim.x) / a.splits;

    // A lane copies 16 bytes of word row lane / 8 of four, so that eight lanes take
    // 128 consecutive bytes; the lane that uses them is (g, t) = (4 columns, row). The
    // place within a row's 128 bytes is permuted by the row, which keeps both the
    // writes and the reads off each other's banks.
    int const fg = lane & 7, ft = lane >> 3;
    uint4* const ring = reinterpret_cast<uint4*>(smem + C::RING * warp) + 8 * t + (g ^ (2 * t));
    uint32_t const ring_u = smem_u32(smem + C::RING * warp) + 16 * (8 * ft + (fg ^ (2 * ft)));
    unsigned char* const mine = smem + C::OFF_D + C::QUAD * (q0 - first);  // digits and offsets, quad by quad
    // Quads are fetched in the order of their use, tile after tile.
    int64_t const w_step = 4 * a.w_r;
    uint32_t const* const w0 = a.w + (16 * static_cast<int64_t>(q0) + ft) * a.w_r + 4 * fg * a.w_n;
    uint32_t const* f_w = w0;
    int f_tile = tile0, f_quad = q0, f_slot = 0, f_cols = 0;  // f_cols: columns from this lane's first on, 0: none
    auto open_tile = [&]() {
        int64_t const col = static_cast<int64_t>(f_tile) * C::COLS;
        f_w = w0 + col * a.w_n;
        f_cols = f_tile < tiles && q0 < q1 ? max(0, static_cast<int>(min(a.N - col, int64_t{C::COLS})) - 4 * fg) : 0;
        f_quad = q0;
    };
    auto fetch = [&]() {
        if (f_tile < tiles && q0 < q1) {
            uint32_t const dst = ring_u + static_cast<uint32_t>(f_slot) * (4 * CT * 512);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool const in = 16 * f_quad + 4 * i + ft < octets;
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    if constexpr (VEC) {
                        if (in && 32 * c < f_cols) copy16(dst + (i * CT + c) * 512, f_w + 32 * c);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (in && 32 * c + e < f_cols) copy4(dst + (i * CT + c) * 512 + 4 * e, f_w + (32 * c + e) * a.w_n);
                    }
                }
                f_w += w_step;
            }
            if (++f_quad == q1) f_tile += stride, open_tile();
        }
        if (++f_slot == C::DEPTH) f_slot = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    open_tile();

    // x's digits: a lane takes an octet of a row at a time, eight steps a warp. First
    // the rows' largest values (the first eight steps' inputs stay in registers, and
    // their loads go out before the weights'), then the digits. Lanes t and t + 1 of
    // a row's four slots hold its high and low digits, so a lane keeps the factor of
    // row t / 2 of its two.
    float down[NT], up[C::ROWS];
    auto load_x = [&](int r, int base, float (&x)[8]) {
        int64_t const m = row0 + r, k = 32 * static_cast<int64_t>(base) + 8 * lane;
        bool const in = m < a.M && k < a.K && base + lane / 4 < s1;
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
    float x[C::ROWS][8];
#pragma unroll
    for (int r = 0; r < C::ROWS; ++r) load_x(r, s0, x[r]);
#pragma unroll
    for (int i = 0; i < C::DEPTH; ++i) fetch();
    {
        unsigned int top[C::ROWS];  // max |x| on the bit patterns: NaN above infinity above every number
        auto raise = [&](float (&y)[8], unsigned int& m) {
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
        };
#pragma unroll
        for (int r = 0; r < C::ROWS; ++r) raise(x[r], top[r] = 0);
        for (int base = s0 + 8; base < s1; base += 8) {
            float y[C::ROWS][8];
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r) load_x(r, base, y[r]);
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r) raise(y[r], top[r]);
        }
#pragma unroll
        for (int r = 0; r < C::ROWS; ++r) {
            unsigned int const m = __reduce_max_sync(0xffffffffu, top[r]);
            // the largest value into [2^29, 2^30): 2^(156 - e), e its biased exponent, where both factors are normal
            int const e = min(max(static_cast<int>(m >> 23), 31), 254);
            up[r] = __int_as_float((283 - e) << 23);
            // NaN and infinity have no whole numbers: the row's sums become NaN
            float const back = m >= 0x7f800000u ? __int_as_float(0x7fffffff) : __int_as_float((e - 29) << 23);
            if ((t >> 1) == (r & 1)) down[r / 2] = back;
        }
    }
    for (int base = s0; base < 4 * q1; base += 8) {
        if (base != s0) {
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r) load_x(r, base, x[r]);
        }
        int const st = base - s0 + (lane >> 2);
        if (st >= 4 * (q1 - q0)) continue;
#pragma unroll
        for (int r = 0; r < C::ROWS; ++r) {
            uint32_t n[8];  // signed base-256 digits: a carry out of the lower bytes, then their signs
#pragma unroll
            for (int i = 0; i < 8; ++i)
                n[i] = (static_cast<uint32_t>(__float2int_rn(x[r][i] * up[r])) + 0x00808080u) ^ 0x00808080u;
            // bytes of elements 0, 2, 4, 6 and 1, 3, 5, 7 (the two masks of a word), digit by digit
            uint32_t d[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t const lo01 = __byte_perm(n[h], n[2 + h], 0x5140), hi01 = __byte_perm(n[h], n[2 + h], 0x7362);
                uint32_t const lo23 = __byte_perm(n[4 + h], n[6 + h], 0x5140), hi23 = __byte_perm(n[4 + h], n[6 + h], 0x7362);
                d[h][0] = __byte_perm(hi01, hi23, 0x7632);
                d[h][1] = __byte_perm(hi01, hi23, 0x5410);
                d[h][2] = __byte_perm(lo01, lo23, 0x7632);
                d[h][3] = __byte_perm(lo01, lo23, 0x5410);
            }
            uint2* const to = reinterpret_cast<uint2*>(mine + C::QUAD * (st / 4)) + ((st % 4) * NT + r / 2) * 32 + (r & 1) * 16 + t;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[4 * j] = make_uint2(d[0][j], d[1][j]);
        }
    }
    __syncwarp();

    // Sums meet their scale after the last step of a group and after the range's
    // last. The bits of such steps in a quad, given the steps left in its group.
    int const left0 = per_group - s0 % per_group;
    auto ends = [&](int quad, int& left) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (--left == 0) m |= 1u << i, left = per_group;
        if (quad + 1 < q1) return m;
        unsigned const last = 1u << (s1 - 1 - 4 * quad);  // steps past K have no group
        return (m & (last - 1u)) | last;
    };
    // 256 times the high plus the low of a pair of digits' sums up to each of these
    // steps: the nibbles' offset of 8, the same for all columns.
    {
        int ones[NT][4], left = left0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) ones[nt][0] = ones[nt][1] = ones[nt][2] = ones[nt][3] = 0;
        for (int quad = q0; quad < q1; ++quad) {
            uint2 const* const dig = reinterpret_cast<uint2 const*>(mine + C::QUAD * (quad - q0)) + lane;
            int* const off = reinterpret_cast<int*>(mine + C::QUAD * (quad - q0) + 4 * NT * 32 * sizeof(uint2));
            unsigned const m = ends(quad, left);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    mma_s8(ones[nt], 0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u, dig[(i * NT + nt) * 32]);
                if (m >> i & 1u) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (g == 0) off[(i * NT + nt) * 4 + t] = 8 * (ones[nt][0] * 256 + ones[nt][1]);
                        ones[nt][0] = ones[nt][1] = ones[nt][2] = ones[nt][3] = 0;
                    }
                }
            }
        }
    }
    __syncwarp();

    int const rows = static_cast<int>(min(static_cast<int64_t>(C::ROWS), a.M - row0));
    int const items = rows * C::COLS, per = (items + a.splits - 1) / a.splits;
    int slot = 0;
    for (int tile = tile0, round = 0; tile < tiles; tile += stride, round ^= 1) {
        int64_t const col0 = static_cast<int64_t>(tile) * C::COLS;
        int const cols = static_cast<int>(min(a.N - col0, int64_t{C::COLS})) - 4 * g;  // from this lane's first on
        float const* ps = a.s + static_cast<int64_t>(s0 / per_group) * a.s_g + (col0 + 4 * g) * a.s_n;
        float acc[NT][CT][4];
        int c[NT][CT][2][4];  // columns 4g + {0, 1} and 4g + {2, 3}: rows g and g + 8 of two products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][k][e] = 0.0f, c[nt][k][0][e] = c[nt][k][1][e] = 0;
        // The scales of a step's group, this lane's columns.
        auto scales = [&](float const* p, float4 (&sc)[CT]) {
#pragma unroll
            for (int k = 0; k < CT; ++k) {
                sc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                float const* pk = p + 32 * k * a.s_n;
                if constexpr (VEC) {
                    if (32 * k < cols) sc[k] = __ldg(reinterpret_cast<float4 const*>(pk));
                } else {
                    if (32 * k < cols) sc[k].x = __ldg(pk);
                    if (32 * k + 1 < cols) sc[k].y = __ldg(pk + a.s_n);
                    if (32 * k + 2 < cols) sc[k].z = __ldg(pk + 2 * a.s_n);
                    if (32 * k + 3 < cols) sc[k].w = __ldg(pk + 3 * a.s_n);
                }
            }
        };
        // Octets past K and columns past N: whatever lies in the ring meets digits of
        // 0, or is not stored.
        auto multiply = [&](uint4 const (&w)[CT], uint2 const (&b)[NT]) {
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t const w0 = h ? w[k].z : w[k].x, w1 = h ? w[k].w : w[k].y;
                    uint32_t const a0 = w0 & 0x0f0f0f0fu, a2 = (w0 >> 4) & 0x0f0f0f0fu;
                    uint32_t const a1 = w1 & 0x0f0f0f0fu, a3 = (w1 >> 4) & 0x0f0f0f0fu;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_s8(c[nt][k][h], a0, a1, a2, a3, b[nt]);
                }
        };
        auto flush = [&](int const* off, float4 const (&sc)[CT]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                int const o = off[4 * nt];
#pragma unroll
                for (int k = 0; k < CT; ++k) {
                    float const f[4] = {sc[k].x, sc[k].y, sc[k].z, sc[k].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int (&q)[4] = c[nt][k][e / 2];
                        int const j = 2 * (e & 1);
                        acc[nt][k][e] = fmaf(static_cast<float>(q[j] * 256 + q[j + 1] - o), f[e], acc[nt][k][e]);
                        q[j] = q[j + 1] = 0;
                    }
                }
            }
        };
        int left = left0;
        for (int quad = q0; quad < q1; ++quad) {
            unsigned const m = ends(quad, left);
            float4 sc[CT];
            if (m != 0u) scales(ps, sc);  // of the first step that needs them; used when the weights have come
            uint2 const* const dig = reinterpret_cast<uint2 const*>(mine + C::QUAD * (quad - q0)) + lane;
            int const* const off = reinterpret_cast<int const*>(mine + C::QUAD * (quad - q0) + 4 * NT * 32 * sizeof(uint2)) + t;
            asm volatile("cp.async.wait_group %0;" ::"n"(C::DEPTH - 1) : "memory");
            __syncwarp();
            uint4 const* const rs = ring + slot * (4 * CT * 32);
            if (++slot == C::DEPTH) slot = 0;
            uint4 w[4][CT];
            uint2 b[4][NT];  // all at once, or with four n-tiles a step's at a time
            auto load_b = [&](int i) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) b[i][nt] = dig[(i * NT + nt) * 32];
            };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int k = 0; k < CT; ++k) w[i][k] = rs[(i * CT + k) * 32];
                if constexpr (NT <= 2) load_b(i);
            }
            __syncwarp();  // the warp has read the quad; its place takes another
            fetch();
            if ((m & 7u) == 0u) {  // groups of 128 inputs or more: no sum ends within the quad
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (NT > 2) load_b(i);
                    multiply(w[i], b[i]);
                }
                if (m != 0u) {
                    flush(off + 12 * NT, sc);
                    ps += a.s_g;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 next[CT];
                    bool const ends_here = m >> i & 1u, another = ends_here && m >> (i + 1) != 0u;
                    if (another) scales(ps + a.s_g, next);
                    if constexpr (NT > 2) load_b(i);
                    multiply(w[i], b[i]);
                    if (!ends_here) continue;
                    flush(off + 4 * NT * i, sc);
                    ps += a.s_g;
                    if (another) {
#pragma unroll
                        for (int k = 0; k < CT; ++k) sc[k] = next[k];
                    }
                }
            }
        }
        // Warps to CTA: high and low digits, the row's factor, then the sums.
        float* const sums = reinterpret_cast<float*>(smem + C::OFF_S) + round * (kWarps * C::ITEMS);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < CT; ++k) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float const low = __shfl_down_sync(0xffffffffu, acc[nt][k][e], 1);
                    v[e] = fmaf(acc[nt][k][e], 65536.0f, low) * down[nt];
                }
                if ((t & 1) == 0)
                    *reinterpret_cast<float4*>(sums + (warp * C::ROWS + 2 * nt + t / 2) * C::COLS + 32 * k + 4 * g) =
                        make_float4(v[0], v[1], v[2], v[3]);
            }
        __syncthreads();
        auto sum_warps = [&](int i) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) v += sums[k * C::ITEMS + i];
            return v;
        };
        auto store = [&](int i, float v) {
            int const r = i / C::COLS;
            int64_t const m = row0 + r, n = col0 + i - r * C::COLS;
            if (n >= a.N) return;
            if (a.bias != nullptr) v += a.bias[n * a.b_n];
            v = activate(v, a.act);
            if (a.res != nullptr) v += a.res[m * a.r_m + n * a.r_n];
            a.y[m * a.y_m + n * a.y_n] = v;
        };
        if (a.splits == 1) {
            for (int i = tid; i < items; i += kThreads) store(i, sum_warps(i));
            continue;
        }
        // CTAs of the cluster: CTA s takes items [s * per, (s + 1) * per) of all of them.
        cg::cluster_group cluster = cg::this_cluster();
        float* const recv = reinterpret_cast<float*>(smem + C::OFF_R) + round * (C::ITEMS + kMaxCluster);
        if (tile == tile0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA runs
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
}

template <int CT, int NT, bool VEC>
int launch(ann_stream stream, LinearQ4Args& a) {
    using C = Q4<CT, NT>;
    auto const kernel = linear_q4_kernel<CT, NT, VEC>;
    static std::mutex mu;
    static std::set<int> ready;  // devices whose kernel attributes are set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "linearQ4: no CUDA device.");
    {
        std::lock_guard<std::mutex> lock(mu);
        if (ready.count(dev) == 0) {
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(C::OFF_D + C::ROOM));
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e != cudaSuccess) return fail(ANN_ECUDA, "linearQ4 setup: %s", cudaGetErrorString(e));
            ready.insert(dev);
        }
    }
    int64_t const tiles = ceil_div(a.N, C::COLS), row_tiles = ceil_div(a.M, C::ROWS), quads = ceil_div(a.K, 128);
    // Splits of the inputs: until every SM has two CTAs, as long as a warp keeps a
    // quad; and as many as x's digits need to fit a CTA.
    int64_t const want = ceil_div(int64_t{2} * sm_count(), tiles * row_tiles);
    int64_t splits = std::max<int64_t>(1, std::min(want, quads / kWarps));
    int64_t const per_quad = static_cast<int64_t>(C::QUAD);
    splits = std::max(splits, ceil_div(quads, C::MAX_QUADS / kMaxCluster));
    splits = std::min<int64_t>(splits, kMaxCluster);
    int64_t const mine = ceil_div(quads, splits) + 1;  // quads of a CTA at most
    size_t const smem = C::OFF_D + static_cast<size_t>(mine * per_quad);
    a.splits = static_cast<int>(splits);
    // As many clusters as fit the GPU at once, each with the same number of tiles or one less.
    int64_t const room = std::max<int64_t>(1, int64_t{sm_count()} * (smem <= (110u << 10) && NT * CT < 4 ? 2 : 1) / (splits * row_tiles));
    int64_t const rounds = ceil_div(tiles, room), clusters = ceil_div(tiles, rounds);
    if (tiles > INT32_MAX || row_tiles > 65535) return fail(ANN_ENOTSUP, "linearQ4: grid too large.");
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * splits), static_cast<unsigned>(row_tiles));
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

// The rows of a CTA: all of them up to eight, fewer where the inputs are so many
// that the digits of eight rows do not fit.
template <int CT>
int launch_rows(ann_stream stream, LinearQ4Args& a, bool vec) {
    int64_t const quads = ceil_div(a.K, 128);
    if (quads > Q4<CT, 1>::MAX_QUADS)
        return fail(ANN_ENOTSUP, "linearQ4: more than %lld inputs.", static_cast<long long>(128 * Q4<CT, 1>::MAX_QUADS));
    if (a.M <= 2 || quads > Q4<CT, 2>::MAX_QUADS) return launch_vec<CT, 1>(stream, a, vec);
    if (a.M <= 4 || quads > Q4<CT, 4>::MAX_QUADS) return launch_vec<CT, 2>(stream, a, vec);
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
    // Few columns: tiles of 32 give twice the CTAs (1024 x 1024, one row: 3.9 us
    // against 4.2); else 64, whose copies, digits and loops serve twice the weights
    // (4096 x 65536: 30 us against 34).
    return a.N < 2048 ? launch_rows<1>(stream, a, vec) : launch_rows<2>(stream, a, vec);
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
