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
#include <array>
#include <map>
#include <mutex>
#include <type_traits>

#include "common.cuh"
#include "overlap.cuh"
#include "pairs.cuh"
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
    int x_vec;       // eight inputs are two aligned 16-byte loads
    int splits;      // CTAs of a cluster that share the inputs
    int share_log2;  // 2^this warps of a CTA share the inputs, the others have columns of their own
    int ends;        // rows of scales that a quad needs at most
    int off_r, off_s, off_d;  // shared memory: the cluster's sums, scales, digits
};

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case ANN_ACT_RELU: return v > 0.0f ? v : 0.0f;
        case ANN_ACT_SILU: return v / (1.0f + expf(-v));
        case ANN_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
        default: return v;
    }
}

// The product in whole numbers. With its top bit flipped a nibble u is u - 8 in two's
// complement; in the upper half of a byte it is the int8 operand 16 (u - 8), so two
// masks (and a shift) unpack the eight of a word. A row of x is rounded to 31 bits of its
// largest value (over the inputs that the CTA shares, or the warp) and cut into four 8-bit digits, and
// mma.sync.m16n8k32 on int8 multiplies, transposed: 16 columns of W by 8 slots,
// the slots being the digits of two rows. The sums are exact in int32, and become fp32
// when their group of inputs or 128 of them end, to meet their
// scale. The order of the summed index is free, so a lane takes the words as a
// 16-byte load gives them, eight inputs (its octet of 32) of four neighbouring
// columns; x's digits are laid out to match.
//
// A CTA stays and takes one set of tiles of 32 CT columns after another. Its warps
// have tiles of their own, or share one, each with inputs of its own (and the CTAs of a
// cluster share them, where columns are few or the digits of all inputs do not fit).
// The digits are prepared once; a warp streams its weights, 128 inputs at a time (a quad
// of products' depth), and their scales through a ring in shared memory (cp.async, on
// across tiles), 4 to 8 KB in flight a warp. The sums of a
// tile meet in shared memory, across a cluster in the CTA that owns a share of the
// columns, which applies bias, activation and residual. One launch, no scratch
// memory, no atomics, a fixed order of sums.
//
// Bound by the weights' bytes, K N (1/2 + 4 / group), for one row; eight rows' products
// take the tensor pipes two thirds of the bytes' time, but with two warps a scheduler
// (256 registers) 0.4 instructions a cycle are issued, and that bounds it. Measured (K x N,
// groups of 128, us, of the bytes' time at the copy rate): one row 4096 x 65536 25.3 (0.87),
// 4096 x 16384 9.3 (0.59), 4096 x 4096 5.2 (0.27: launch, digits, one turn of memory); eight
// rows 4096 x 16384, groups of 64, 18.5 (0.32), 4096 x 65536 56 (0.42). The weights are read
// once for every eight rows: 4096 x 16384, 16 rows 28.0, 32 50.9, 64 96.3.
constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 16;
constexpr size_t kMaxSmem = 227 * 1024;

// The int32 sums start at the bits of 1.5 * 2^23: with less than 2^22 added (128
// products of at most 128 * 128), the bits are those of the fp32 value 1.5 * 2^23 +
// sum, and no conversion is needed.
constexpr int kStartBits = 0x4b400000;

// Shared memory: rings [kWarps][DEPTH quads][4][CT][32] uint4, two buffers of sums
// [kWarps][ROWS][COLS]; by the call, two of the cluster's [per * splits], scales
// [kWarps][DEPTH + 1][ends][COLS] and, per quad of the CTA, digits uint2 [4][NT][32].
template <int CT, int NT, int QUADS = 4 / CT>
struct Q4 {
    static constexpr int COLS = 32 * CT, ROWS = 2 * NT, ITEMS = ROWS * COLS;
    static constexpr int DEPTH = QUADS;                              // quads in flight a warp
    static constexpr size_t RING = size_t{16} * DEPTH * 4 * CT * 32;  // of a warp
    static constexpr size_t OFF_S = RING * kWarps;
    static constexpr size_t FIXED = OFF_S + sizeof(float) * 2 * kWarps * ITEMS;
    static constexpr size_t QUAD = size_t{4} * NT * 32 * sizeof(uint2);
    static constexpr size_t scales(int ends) { return sizeof(float) * kWarps * (DEPTH + 1) * ends * COLS; }
    static constexpr size_t received(int columns) { return sizeof(float) * 2 * (ROWS * columns + kMaxCluster); }
    // Quads of inputs whose digits fit a CTA at the least.
    static constexpr int64_t LEAST = (kMaxSmem - FIXED - scales(4) - received(COLS)) / QUAD;
};

// c += a b, or c = start + a b: int8 products of depth 32, exact in int32.
template <bool FRESH>
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    if constexpr (FRESH)
        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y), "r"(kStartBits));
    else
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
// rows a CTA); VEC: words and scales of four columns are one aligned load; ENDS: groups
// that end in a quad, 1 (groups of 128, 256, ..), 2 (64), 4 (32) or 0 (any). Code for one
// kind of group only is a third of the instructions to fetch (4096 x 65536, one row, groups
// of 128, 64 and 32: 25.4, 27.0 and 29.9 us against 28.0, 28.3 and 33.6).
template <typename C, int CT, int NT, bool VEC, int ENDS>
__global__ void __launch_bounds__(kThreads, NT * CT >= 4 ? 1 : 2) linear_q4_kernel(LinearQ4Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    int const tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int const split = static_cast<int>(blockIdx.x) % a.splits;
    if (a.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // "this CTA runs"
    int64_t const row0 = static_cast<int64_t>(blockIdx.y) * C::ROWS;
    // the CTA's quads of 128 inputs [first, last), the warp's [q0, q1), in steps of 32;
    // `across` warps side by side have tiles of their own, `share` the same one
    int const quads = static_cast<int>((a.K + 127) / 128), steps = static_cast<int>((a.K + 31) / 32);
    int const first = static_cast<int>(static_cast<int64_t>(quads) * split / a.splits);
    int const last = static_cast<int>(static_cast<int64_t>(quads) * (split + 1) / a.splits);
    int const share = 1 << a.share_log2, across_log2 = 3 - a.share_log2, across = 1 << across_log2;
    int const part = warp >> across_log2, mine = warp & (across - 1);
    int const q0 = first + ((last - first) * part >> a.share_log2), q1 = first + ((last - first) * (part + 1) >> a.share_log2);
    int const octets = static_cast<int>(a.K / 8), per_group = a.group / 32, groups = (steps + per_group - 1) / per_group;
    int const tiles = static_cast<int>((a.N + C::COLS - 1) / C::COLS);
    int const sets = (tiles + across - 1) >> across_log2;  // a CTA's tiles at a time
    int const set0 = static_cast<int>(blockIdx.x) / a.splits, stride = static_cast<int>(gridDim.x) / a.splits;

    // A lane copies 16 bytes of word row lane / 8 of four, so that eight lanes take
    // 128 consecutive bytes; the lane that uses them is (g, t) = (4 columns, row). The
    // place within a row's 128 bytes is permuted by the row, which keeps both the
    // writes and the reads off each other's banks.
    int const fg = lane & 7, ft = lane >> 3;
    uint4* const ring = reinterpret_cast<uint4*>(smem + C::RING * warp) + 8 * t + (g ^ (2 * t));
    uint32_t const ring_u = smem_u32(smem + C::RING * warp) + 16 * (8 * ft + (fg ^ (2 * ft)));
    int const place_size = a.ends * C::COLS;  // floats
    float* const scale_ring = reinterpret_cast<float*>(smem + a.off_s) + warp * (C::DEPTH + 1) * place_size;
    uint32_t const scale_ring_u = smem_u32(scale_ring);
    // Sums meet their scale after the last step of a group and of a quad. The bits of
    // such steps (ENDS == 0), given the steps left in the group; `passed`: groups that end.
    int const left0 = per_group - 4 * q0 % per_group;
    auto ends = [&](int quad, int& left, int& passed) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (--left == 0) m |= 1u << i, left = per_group;
        passed = __popc(m);
        unsigned const end = 1u << min(3, steps - 1 - 4 * quad);  // steps past K have no group
        return (m & (end - 1u)) | end;
    };
    // Quads are fetched in the order of their use, tile after tile, each with the
    // rows of scales that its sums meet. Scales have one place more than weights, as
    // they are read until the quad's end, its weights only at its start.
    int64_t const w_step = 4 * a.w_r;
    uint32_t const* const w0 = a.w + (16 * static_cast<int64_t>(q0) + ft) * a.w_r + 4 * fg * a.w_n;
    uint32_t const* f_w = w0;
    float const* f_s = a.s;
    int f_tile = set0 * across + mine, f_quad = q0, f_slot = 0, f_place = 0, f_cols = 0, f_left = left0;  // f_cols: columns of the tile
    auto open_tile = [&]() {
        int64_t const col = static_cast<int64_t>(f_tile) * C::COLS;
        f_w = w0 + col * a.w_n;
        f_s = a.s + static_cast<int64_t>(4 * q0 / per_group) * a.s_g + col * a.s_n;
        f_cols = static_cast<int>(min(a.N - col, int64_t{C::COLS}));
        f_quad = q0;
        f_left = left0;
    };
    auto fetch = [&]() {
        if (f_tile < tiles && q0 < q1) {
            uint32_t const dst = ring_u + static_cast<uint32_t>(f_slot) * (4 * CT * 512);
            int const from = f_cols - 4 * fg;  // columns from this lane's first on
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool const in = 16 * f_quad + 4 * i + ft < octets;
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    if constexpr (VEC) {
                        if (in && 32 * c < from) copy16(dst + (i * CT + c) * 512, f_w + 32 * c);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (in && 32 * c + e < from) copy4(dst + (i * CT + c) * 512 + 4 * e, f_w + (32 * c + e) * a.w_n);
                    }
                }
                f_w += w_step;
            }
            // rows of scales; of groups that K leaves out the last one's, which meets sums of 0
            int passed = ENDS, n = ENDS, most = 3;
            if constexpr (ENDS == 0) {
                n = __popc(ends(f_quad, f_left, passed));
            } else if constexpr (ENDS == 1) {
                passed = (f_left -= 4) == 0;
                if (passed) f_left = per_group;
            } else {
                most = groups - 1 - ENDS * f_quad;
            }
            uint32_t const dst_s = scale_ring_u + static_cast<uint32_t>(f_place * place_size) * 4;
#pragma unroll
            for (int e = 0; e < CT; ++e) {
                int const i = lane + 32 * e, r = i / (8 * CT), c = 4 * (i % (8 * CT));
                float const* const p = f_s + min(r, most) * a.s_g + c * a.s_n;
                if constexpr (VEC) {
                    if (r < n && c < f_cols) copy16(dst_s + 16 * i, p);
                } else {
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        if (r < n && c + d < f_cols) copy4(dst_s + 16 * i + 4 * d, p + d * a.s_n);
                }
            }
            f_s += passed * a.s_g;
            if (++f_quad == q1) f_tile += stride * across, open_tile();
        }
        if (++f_slot == C::DEPTH) f_slot = 0;
        if (++f_place == C::DEPTH + 1) f_place = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    open_tile();
    prior_kernels_done();

    // x's digits: every warp prepares an eighth of the CTA's quads (its own, if all
    // warps share a tile). A lane takes an octet of a row at a time, eight steps a warp. First
    // the rows' largest values (the first eight steps' inputs stay in registers, and
    // their loads go out before the weights'), then the digits. Lanes t and t + 1 of
    // a row's four slots hold its high and low digits, so a lane keeps the factor of
    // row t / 2 of its two.
    int const s0 = 4 * (first + ((last - first) * warp >> 3)), s_end = 4 * (first + ((last - first) * (warp + 1) >> 3));
    int const s1 = min(s_end, steps);
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
        for (int r = 0; r < C::ROWS; ++r) top[r] = __reduce_max_sync(0xffffffffu, top[r]);
        if (across > 1) {  // digits of one warp meet weights of another: one factor for all
            unsigned int* const all = reinterpret_cast<unsigned int*>(smem + C::OFF_S);
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r)
                if (lane == 0) all[warp * C::ROWS + r] = top[r];
            __syncthreads();
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r) top[r] = __reduce_max_sync(0xffffffffu, all[(lane & 7) * C::ROWS + r]);
        }
#pragma unroll
        for (int r = 0; r < C::ROWS; ++r) {
            unsigned int const m = top[r];
            // the largest value into [2^29, 2^30): 2^(156 - e), e its biased exponent, where both factors are normal
            int const e = min(max(static_cast<int>(m >> 23), 31), 254);
            up[r] = __int_as_float((283 - e) << 23);
            // NaN and infinity have no whole numbers: the row's sums become NaN
            float const back = m >= 0x7f800000u ? __int_as_float(0x7fffffff) : __int_as_float((e - 29) << 23);
            if ((t >> 1) == (r & 1)) down[r / 2] = back;
        }
    }
    for (int base = s0; base < s_end; base += 8) {
        if (base != s0) {
#pragma unroll
            for (int r = 0; r < C::ROWS; ++r) load_x(r, base, x[r]);
        }
        int const st = base - 4 * first + (lane >> 2);
        if (st >= s_end - 4 * first) continue;
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
            uint2* const to = reinterpret_cast<uint2*>(smem + a.off_d + C::QUAD * (st / 4)) + ((st % 4) * NT + r / 2) * 32 + (r & 1) * 16 + t;
#pragma unroll
            for (int j = 0; j < 4; ++j) to[4 * j] = make_uint2(d[0][j], d[1][j]);
        }
    }
    if (across > 1)
        __syncthreads();
    else
        __syncwarp();

    unsigned char const* const digits = smem + a.off_d + C::QUAD * (q0 - first);
    int const rows = static_cast<int>(min(static_cast<int64_t>(C::ROWS), a.M - row0));
    int const width_log2 = (CT == 1 ? 5 : 6) + across_log2, items = rows << width_log2;  // of a set
    int const per = (items + a.splits - 1) / a.splits;
    int slot = 0, place = 0;
    pair_t const start = pair(-12582912.0f, -12582912.0f);
    for (int set = set0, round = 0; set < sets; set += stride, round ^= 1) {
        pair_t acc[NT][CT][4];  // a pair of digits, high and low, of columns 4g ..
        int c[NT][CT][2][4];  // columns 4g + {0, 1} and 4g + {2, 3}: rows g and g + 8 of two products
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][k][e] = pair(0.0f, 0.0f);
        // Octets past K and columns past N: whatever lies in the ring meets digits of
        // 0, or is not stored. FRESH: the first product of a sum.
        auto multiply = [&]<bool FRESH>(std::bool_constant<FRESH>, uint4 const (&w)[CT], uint2 const (&b)[NT]) {
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t const w0 = h ? w[k].z : w[k].x, w1 = h ? w[k].w : w[k].y;
                    uint32_t const a0 = (w0 << 4 ^ 0x80808080u) & 0xf0f0f0f0u, a2 = (w0 ^ 0x80808080u) & 0xf0f0f0f0u;
                    uint32_t const a1 = (w1 << 4 ^ 0x80808080u) & 0xf0f0f0f0u, a3 = (w1 ^ 0x80808080u) & 0xf0f0f0f0u;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_s8<FRESH>(c[nt][k][h], a0, a1, a2, a3, b[nt]);
                }
        };
        // Sums to fp32, with the scales sc[8 k] of column word k.
        auto flush = [&](float4 const* sc) {
#pragma unroll
            for (int k = 0; k < CT; ++k) {
                float4 const s4 = sc[8 * k];
                pair_t const f[4] = {pair(s4.x, s4.x), pair(s4.y, s4.y), pair(s4.z, s4.z), pair(s4.w, s4.w)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        int const (&q)[4] = c[nt][k][e / 2];
                        int const j = 2 * (e & 1);
                        acc[nt][k][e] = fma2(add2(pair(__int_as_float(q[j]), __int_as_float(q[j + 1])), start), f[e], acc[nt][k][e]);
                    }
            }
        };
        bool const given = (set << across_log2) + mine < tiles;
        int left = left0;
        for (int quad = q0; quad < q1 && given; ++quad) {
            uint2 const* const dig = reinterpret_cast<uint2 const*>(digits + C::QUAD * (quad - q0)) + lane;
            asm volatile("cp.async.wait_group %0;" ::"n"(C::DEPTH - 1) : "memory");
            __syncwarp();
            uint4 const* const rs = ring + slot * (4 * CT * 32);
            if (++slot == C::DEPTH) slot = 0;
            float4 const* sc = reinterpret_cast<float4 const*>(scale_ring + place * place_size) + g;
            if (++place == C::DEPTH + 1) place = 0;
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
            constexpr std::true_type fresh{};
            constexpr std::false_type more{};
            if constexpr (ENDS > 0) {
                constexpr int LONG = 4 / ENDS;  // steps of a sum
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (NT > 2) load_b(i);
                    if (i % LONG == 0) multiply(fresh, w[i], b[i]);
                    else multiply(more, w[i], b[i]);
                    if (i % LONG == LONG - 1) flush(sc + i / LONG * (8 * CT));
                }
            } else {
                int passed;
                unsigned const m = ends(quad, left, passed);
                bool begins = true;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (NT > 2) load_b(i);
                    if (begins) multiply(fresh, w[i], b[i]);
                    else multiply(more, w[i], b[i]);
                    begins = m >> i & 1u;
                    if (begins) flush(sc), sc += 8 * CT;
                }
            }
        }
        // Warps to CTA: high and low digits, the row's factor (and the 16 of the
        // operands), then the sums.
        float* const sums = reinterpret_cast<float*>(smem + C::OFF_S) + round * (kWarps * C::ITEMS);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < CT; ++k) {
                float v[4];
                float const unit = (t & 1 ? 0.0625f : 4096.0f) * down[nt];  // first of all, so that nothing overflows on the way
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float2 const d = unpair(acc[nt][k][e]);
                    float const two = fmaf(d.x, 256.0f * unit, d.y * unit);
                    v[e] = two + __shfl_down_sync(0xffffffffu, two, 1);
                }
                if ((t & 1) == 0)
                    *reinterpret_cast<float4*>(sums + (warp * C::ROWS + 2 * nt + t / 2) * C::COLS + 32 * k + 4 * g) =
                        make_float4(v[0], v[1], v[2], v[3]);
            }
        __syncthreads();
        // item i of a set: row i >> width_log2, then the columns of its tiles
        auto sum_warps = [&](int i) {
            int const r = i >> width_log2, col = i & ((1 << width_log2) - 1);
            float const* p = sums + (col / C::COLS * C::ROWS + r) * C::COLS + col % C::COLS;
            float v = 0.0f;
            for (int k = 0; k < share; ++k) v += p[k * (C::ITEMS << across_log2)];
            return v;
        };
        auto store = [&](int i, float v) {
            int64_t const m = row0 + (i >> width_log2), n = (static_cast<int64_t>(set) << width_log2) + (i & ((1 << width_log2) - 1));
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
        float* const recv = reinterpret_cast<float*>(smem + a.off_r) + round * ((C::ROWS << width_log2) + kMaxCluster);
        if (set == set0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA runs
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

// Clusters of 1 .. kMaxCluster CTAs that the device holds at once, with one and two
// CTAs an SM.
using Room = std::array<std::array<int, kMaxCluster + 1>, 2>;
constexpr size_t kHalfSmem = 113 * 1024;

template <typename C, int CT, int NT, bool VEC, int ENDS>
int launch(ann_stream stream, LinearQ4Args& a) {
    auto const kernel = linear_q4_kernel<C, CT, NT, VEC, ENDS>;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attrs[2] = {{}, overlapping()}, &attr = attrs[0];
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.blockDim = dim3(kThreads);
    cfg.attrs = attrs;
    cfg.numAttrs = 2;
    static std::mutex mu;
    static std::map<int, Room> rooms;  // devices whose kernel attributes are set
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "linearQ4: no CUDA device.");
    Room const* room = nullptr;
    {
        std::lock_guard<std::mutex> lock(mu);
        auto it = rooms.find(dev);
        if (it == rooms.end()) {
            Room r{};
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxSmem));
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            for (int two = 0; two < 2; ++two)
                for (int n = 1; n <= kMaxCluster && e == cudaSuccess; ++n) {
                    attr.val.clusterDim.x = static_cast<unsigned>(n);
                    cfg.gridDim = dim3(static_cast<unsigned>(n));
                    cfg.dynamicSmemBytes = two ? kHalfSmem : kMaxSmem;
                    e = cudaOccupancyMaxActiveClusters(&r[two][n], kernel, &cfg);
                }
            if (e != cudaSuccess) return fail(ANN_ECUDA, "linearQ4 setup: %s", cudaGetErrorString(e));
            it = rooms.emplace(dev, r).first;
        }
        room = &it->second;
    }
    int64_t const tiles = ceil_div(a.N, C::COLS), row_tiles = ceil_div(a.M, C::ROWS), quads = ceil_div(a.K, 128);
    if (tiles > INT32_MAX || row_tiles > 65535) return fail(ANN_ENOTSUP, "linearQ4: grid too large.");
    a.ends = a.group == 32 ? 4 : a.group % 128 == 0 ? 1 : 2;
    // How many warps of a CTA and CTAs of a cluster share the inputs: the least of
    // these estimates (us, fitted to measured shapes). A quad takes a warp its memory's latency
    // with two in flight, or its turn among the SM's warps; preparing a quad's digits,
    // and what a set of tiles costs to sum and store, count beside it. (On thirteen shapes at
    // up to 36 choices each the estimate's is within 3 % of the best; us of it, of all eight
    // warps to a tile, of a tile a warp, each with its best cluster: 8 x 4096 x 16384 18.5,
    // 22.6, 19.3; 1 x 4096 x 4096 5.1, 5.1, 6.5; 1 x 4096 x 65536 24.9, 26.3, 25.0; 1 x 16384 x
    // 4096 9.2, 10.1, 13.9.)
    size_t smem = 0;
    int64_t clusters = 0;
    double best = 1e300;
    for (int share_log2 = 3; share_log2 >= 0; --share_log2) {
        int const across = kWarps >> share_log2;
        size_t const fixed = C::FIXED + C::scales(a.ends);
        for (int splits = 1; splits <= kMaxCluster; ++splits) {
            int64_t const in_cta = ceil_div(quads, splits), in_warp = ceil_div(in_cta, int64_t{1} << share_log2);
            size_t const recv = splits > 1 ? C::received(C::COLS * across) : 0;
            size_t const need = fixed + recv + static_cast<size_t>(in_cta) * C::QUAD;
            if (need > kMaxSmem || (splits > 1 && splits > quads)) continue;
            int const most = (*room)[need <= kHalfSmem][splits];
            if (most == 0) continue;
            // as many clusters as fit the GPU at once, each with the same number of sets or one less
            int64_t const at_once = std::max<int64_t>(1, most / row_tiles), sets = ceil_div(tiles, across);
            int64_t const rounds = ceil_div(sets, at_once), used = ceil_div(sets, rounds);
            int const load = need <= kHalfSmem && NT * CT < 4 && used * row_tiles > (*room)[0][splits] ? 2 : 1;  // CTAs of an SM
            double const quad = std::max(0.8 + 0.1 * a.ends, kWarps * load * (0.017 + 0.0275 * NT + 0.003 * a.ends) * CT);
            double const prepare = (0.3 + 0.1 * NT) * load * static_cast<double>(in_cta) / kWarps;
            double const finish = 1.5 + 0.06 * NT * CT * across * load + (splits > 1 ? 0.4 + 0.05 * splits : 0.0);
            double const cost = prepare + static_cast<double>(rounds) * (static_cast<double>(in_warp) * quad + finish);
            if (cost >= best) continue;
            best = cost;
            a.share_log2 = share_log2;
            a.splits = splits;
            a.off_r = static_cast<int>(C::FIXED);
            a.off_s = static_cast<int>(C::FIXED + recv);
            a.off_d = static_cast<int>(fixed + recv);
            smem = need;
            clusters = used;
        }
    }
    if (clusters == 0) return fail(ANN_ENOTSUP, "linearQ4: no cluster holds the inputs.");
    attr.val.clusterDim.x = static_cast<unsigned>(a.splits);
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * a.splits), static_cast<unsigned>(row_tiles));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = as_stream(stream);
    cudaLaunchKernelEx(&cfg, kernel, a);
    return check_launch("linearQ4");
}

template <int CT, int NT, int QUADS = 4 / CT>
int launch_vec(ann_stream stream, LinearQ4Args& a, bool vec) {
    using C = Q4<CT, NT, QUADS>;
    if (!vec) return launch<C, CT, NT, false, 0>(stream, a);
    if (a.group % 128 == 0) return launch<C, CT, NT, true, 1>(stream, a);
    if (a.group == 64) return launch<C, CT, NT, true, 2>(stream, a);
    if (a.group == 32) return launch<C, CT, NT, true, 4>(stream, a);
    return launch<C, CT, NT, true, 0>(stream, a);
}

// The rows of a CTA: all of them up to eight, fewer where the inputs are so many
// that the digits of eight rows do not fit; at last with a shorter ring beside them.
template <int CT>
int launch_rows(ann_stream stream, LinearQ4Args& a, bool vec) {
    using Longest = Q4<1, 1, 2>;
    int64_t const quads = ceil_div(a.K, 128);
    if (quads > kMaxCluster * Longest::LEAST)
        return fail(ANN_ENOTSUP, "linearQ4: more than %lld inputs.", static_cast<long long>(128 * kMaxCluster * Longest::LEAST));
    if (quads > kMaxCluster * Q4<CT, 1>::LEAST) return launch_vec<1, 1, 2>(stream, a, vec);
    if (a.M <= 2 || quads > kMaxCluster * Q4<CT, 2>::LEAST) return launch_vec<CT, 1>(stream, a, vec);
    if (a.M <= 4 || quads > kMaxCluster * Q4<CT, 4>::LEAST) return launch_vec<CT, 2>(stream, a, vec);
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
    ANN_TRY(to_dims_flat(p_v, sizeof(uint32_t), what, p));
    ANN_TRY(to_dims_flat(s_v, sizeof(float), what, s));
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
    ANN_TRY(to_dims_flat(x_v, sizeof(float), "linearQ4 input", x));
    ANN_TRY(check_packed("linearQ4", p_v, s_v, group, p, s));
    ANN_TRY(to_dims_flat(y_v, sizeof(float), "linearQ4 output", y));
    if (act < ANN_ACT_NONE || act > ANN_ACT_GELU) return fail(ANN_EINVAL, "linearQ4: unknown activation %d.", act);
    if (x.rank != 2 || y.rank != 2 || x.ext[1] != 8 * p.ext[0] || y.ext[0] != x.ext[0] || y.ext[1] != p.ext[1])
        return fail(ANN_EINVAL, "linearQ4 shape mismatch.");
    if (!writable(y)) return fail(ANN_EINVAL, "linearQ4: an output axis has a zero pitch.");
    LinearQ4Args a{};
    if (b_v != nullptr) {
        ANN_TRY(to_dims_flat(b_v, sizeof(float), "linearQ4 bias", b));
        if (b.rank != 1 || b.ext[0] != y.ext[1]) return fail(ANN_EINVAL, "linearQ4 expects a 1D bias matching the output.");
        a.bias = static_cast<const float*>(b.data);
        a.b_n = b.str[0];
    }
    if (r_v != nullptr) {
        ANN_TRY(to_dims_flat(r_v, sizeof(float), "linearQ4 residual", r));
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
    // Few columns: tiles of 32 give twice the CTAs (1024 x 1024: 3.0 us against 3.6,
    // eight rows 5.4 against 6.2); else 64, whose copies, digits and loops serve twice
    // the weights (4096 x 65536: 25.4 us against 26.2; 4096 x 2048: 4.5 against 4.8).
    return a.N < 2048 ? launch_rows<1>(stream, a, vec) : launch_rows<2>(stream, a, vec);
}

int pack_q4(ann_stream stream, const ann_view* w_v, const ann_view* p_v, const ann_view* s_v, uint32_t group) {
    Dims w, p, s;
    ANN_TRY(to_dims_flat(w_v, sizeof(float), "packWeightQ4 weight", w));
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
