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
#include <array>
#include <cmath>
#include <map>
#include <mutex>
#include <set>

#include "common.cuh"
#include "overlap.cuh"
#include "pairs.cuh"
#include "reduce.cuh"
#include "tma.cuh"

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
    int splits;         // CTAs of a cluster that share a KV head's keys
    float* parts;       // of the even shares: [2 * gridDim.x][ROWS * D], then [2 * gridDim.x][2][ROWS]
    int block_shift, causal;
    float scale;
};

// How the products are formed. q.k in whole numbers: a row of q is rounded to 31 bits
// of its largest value and cut into four 8-bit digits, so that mma.sync.m16n8k32 on
// int8 multiplies the cache's bytes as they are, and the sums are exact. With up to
// four query rows of a KV head (R = 4) one product holds all their digits; with up to
// eight one holds the high two, another the low two.
// p.v in halves: a cached value is exact in fp16, a probability (times V's scale, relative
// to the tile's largest of both) is the sum of two fp16 parts (22 bits), and
// mma.sync.m16n8k16 adds the exact products in fp32, both parts of eight rows in one
// product, from a fresh accumulator for each tile, so that no sum of more than KT
// products is left to the tensor core's own rounding. Every key has to keep its own
// bits: a column of V may be 0 wherever the probabilities are large. The low part is held
// 2^13 times finer than the high one, so 22 bits reach 2^-30 (20 nats) below the
// tile's largest. Tiles with scores further apart are marked, and where a sum is so small that
// what they lost may show, they are multiplied once more. (8 x 2048 keys, 32 heads:
// 27.6 us for scores of 2 and of 4.5 nats' standard deviation, 44 for 9; 1 x 131072, eight rows:
// 37.4, 39 and 50.)
// (Digits for p.v too, against one reference for the row, would be 2 us less for 8 x 2048
// keys, but hold every key to the same step, 2^-25 of the largest.)
// (On this GPU an int8 product of depth 32 and an fp16 one of depth 16 take the same
// time, 2.1 cycles of an SM: 8 KB of cache cost 64 of them, 0.4 of the time that HBM
// takes to deliver it; 48 with R = 4.)
//
// How the cache reaches the fragments. The order of the summed index and of the
// output columns of a matrix product is free as long as both operands agree, so
// a lane takes whole 16-byte pieces: of one key's row for q.k (four lanes cover a
// key), of four keys at the same elements for p.v (eight lanes cover a row). No
// transposition is needed. Every warp streams tiles of KT keys of its own through
// a ring of two tiles in shared memory (cp.async, 16 bytes a lane, rows of 128
// bytes coalesced), one tile ahead of the one it works on: 8 to 16 KB in flight
// a warp, 12 warps an SM, where HBM's latency asks for 40 KB an SM. The pieces
// are placed so that both kinds of reads are free of bank conflicts.
//
// Every warp keeps a running maximum and sum per row (base 2). Warps meet in
// shared memory; the CTAs of a cluster (the key range's splits) send their parts into
// each other's shared memory, where each CTA sums its share of the output: one cluster
// barrier, no scratch memory, no atomics, one launch, and a fixed order of sums. Long
// caches go in even shares over all CTAs instead, with a second kernel for the parts.
//
// Bound by the cache's bytes, 2 D a key and KV head. Measured (us, of the bytes' time
// at the copy rate): 16 x 32768 keys, 64/8 heads 174 (0.96; 213 with launches back to
// back for seconds, when the power limit lowers the clock), 8 x 2048, 32/32 27.8 (0.75),
// 1 x 131072, 32/4 37.5 (0.55: ten rounds of tiles a warp where 9.2 would do, and 5 us
// for the merge), 12 x 4096 of 64, four tokens, 16/4 12.7 (0.16: the start, and 8 warps'
// chains of product, maximum, exponential, product), 1 x 300, 32/8 5.3 (launch, two turns
// of memory, the cluster's barrier).
constexpr int kMaxCluster = 16;
constexpr int kMaxShares = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFiner = 1.0f / 2251799813685248.0f, kSmall = 1.0f / 65536.0f;  // 2^-51, 2^-16: see rest

template <int D, int R, int W>
struct Q8 {
    static constexpr int THREADS = 32 * W;
    static constexpr int MT = R == 16 ? 2 : 1;     // groups of eight rows
    static constexpr int KT = D <= 128 ? 32 : 16;  // keys per tile of a warp
    static constexpr int ROWS = R;                 // query rows of a CTA
    static constexpr int KS = D / 32;              // k32 steps of q.k
    static constexpr int QT = R == 4 ? 1 : 2;      // products that hold a row's digits
    static constexpr int NK = KT / 8;              // n8 tiles of keys
    static constexpr int KV = KT / 16;             // k16 steps of p.v, groups of 16 keys
    static constexpr int VW = D / 32;              // words of V per lane and key
    static constexpr int KW = D / 16;              // words of K per lane and key
    // q's fragments in registers, or read again for each tile (in registers 16 x 32768 keys of
    // 128, eight rows a head: 180 us against 171, 9 x 16576: 59 against 56)
    static constexpr bool QREG = MT * KS <= 2;
    static constexpr int TILE = KT * D;            // bytes of a tile of K or V
    static constexpr int RING = 4 * TILE;          // K, V, K, V of a warp; its output rows at the end
    static constexpr int PER_SM = R <= 8 && D <= 128 ? 3 : 2;  // CTAs, by registers
    static constexpr size_t OFF_Q = size_t{1} * RING * W;                      // uint4 [MT][KS][QT][32]
    static constexpr size_t OFF_R = OFF_Q + size_t{16} * MT * KS * QT * 32;    // float4 [ROWS * D / 4 + kMaxCluster]
    static constexpr size_t OFF_ML = OFF_R + sizeof(float) * (ROWS * D + 4 * kMaxCluster);  // float [2][W][ROWS]
    static constexpr size_t OFF_F = OFF_ML + sizeof(float) * 2 * W * ROWS;     // float [ROWS]: score factors
    static constexpr size_t OFF_X = OFF_F + sizeof(float) * ROWS;              // float [kMaxCluster][2][ROWS]: max, sum
    static constexpr size_t SMEM = OFF_X + sizeof(float) * kMaxCluster * 2 * ROWS;
    static_assert(RING >= static_cast<int>(sizeof(float)) * ROWS * D, "a warp's output rows fit its ring");
    // 16-byte piece c of row r of a tile, with the pieces of a 128-byte line
    // permuted: K is read by 8 lanes as two rows x every other piece (or four), V
    // as every other row of 8 x two neighbouring pieces (or halves of them).
    static __device__ __forceinline__ uint32_t place(int r, int c) {
        if constexpr (D == 64) {
            int const line = r >> 1, q = (r & 1) * 4 + c;
            return line * 128 + ((q ^ ((line & 1) << 2) ^ (line & 2)) << 4);
        } else {
            return r * D + (c >> 3) * 128 + (((c & 7) ^ (r & 7)) << 4);
        }
    }
    // Piece i of lane t for q.k.
    static __device__ __forceinline__ int piece(int i, int t) { return D == 64 ? t : 8 * (i >> 1) + 2 * t + (i & 1); }
};

// c += a b (or c = a b): fp16 products of depth 16, summed in fp32.
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t const (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t const (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// int8 products of depth 32, exact in int32.
__device__ __forceinline__ void mma_s8(int (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int (&c)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(0));
}

// 2^x for x <= 0; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_neg(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two unsigned bytes u (= n + 128) of w picked by `sel` as fp16 whole numbers n:
// 0x6400 | u is 1024 + u, and 1024 + 128 is taken off, all exact.
__device__ __forceinline__ uint32_t halves_of(uint32_t w, uint32_t sel) {
    uint32_t const biased = __byte_perm(w, 0x64646464u, sel);
    __half2 const h = __hsub2(*reinterpret_cast<__half2 const*>(&biased), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<uint32_t const*>(&h);
}

// x, y -> their fp16 parts, high and low, each as a pair; the low ones in units 2^13 times
// finer, so that they too are normal numbers: below 2^15 for x and y below 2^14.
constexpr float kLowUnit = 1.0f / 8192.0f;
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    __half2 const h = __floats2half2_rn(x, y);
    float2 const f = __half22float2(h);
    __half2 const l = __floats2half2_rn((x - f.x) * (1.0f / kLowUnit), (y - f.y) * (1.0f / kLowUnit));
    hi = *reinterpret_cast<uint32_t const*>(&h);
    lo = *reinterpret_cast<uint32_t const*>(&l);
}

// What two parts leave of x below 2^-16, in units 2^51 times finer: exact, and at most 2^13.
__device__ __forceinline__ float rest(float x) {
    float const r = x - __half2float(__float2half_rn(x));
    float const l = __half2float(__float2half_rn(r * (1.0f / kLowUnit)));
    return fabsf(x) < kSmall ? fmaf(l, -kLowUnit, r) * (1.0f / kFiner) : 0.0f;
}

// 16 bytes from global to shared memory, asynchronously, in the thread's open group.
__device__ __forceinline__ void copy16(uint32_t dst, const int8_t* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest N groups have landed, for every lane of the warp.
template <int N>
__device__ __forceinline__ void copies_landed() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
    __syncwarp();
}

// 2^(e - 127) for a biased exponent e in [1, 254].
__device__ __forceinline__ float pow2_biased(int e) { return __int_as_float(e << 23); }

// ---- even shares of all keys ----------------------------------------------------
// The tiles of every KV head of every sequence in one row, KV heads (and row
// tiles) of a sequence one after another; CTA c of G takes tiles [cut(c),
// cut(c + 1)), whole rounds of its W warps. Lengths are known on the device only,
// so both kernels walk them.
struct Shares {
    int total, W, q, rem;  // the first rem CTAs take q + 1 rounds, the others q
    __device__ Shares(int total, int G, int W) : total(total), W(W) {
        int const rounds = (total + W - 1) / W;
        q = rounds / G;
        rem = rounds - q * G;
    }
    __device__ int cut(int c) const { return min(total, W * (c * q + min(c, rem))); }
    // The CTA whose share tile p < total lies in.
    __device__ int owner(int p) const {
        int const r = p / W, wide = rem * (q + 1);
        return r < wide ? r / (q + 1) : rem + (r - wide) / q;
    }
};

// Keys of sequence b.
__device__ __forceinline__ int64_t keys_of(DecodeQ8Args const& a, int64_t b) {
    if (a.lengths == nullptr) return a.cap;
    return min(a.cap, max(int64_t{0}, static_cast<int64_t>(a.lengths[b * a.len_s])));
}

// Tiles of the first `stop` sequences of one KV head and row tile (each warp by itself).
template <int KT>
__device__ __forceinline__ int tiles_before(DecodeQ8Args const& a, int64_t stop) {
    int sum = 0;
    for (int64_t b = threadIdx.x & 31; b < stop; b += 32) sum += static_cast<int>((keys_of(a, b) + KT - 1) / KT);
    return warp_sum(sum);
}
// The sequence that holds tile p of one KV head's row, and its first tile.
template <int KT>
__device__ __forceinline__ int64_t sequence_of(DecodeQ8Args const& a, int p, int& first) {
    int const lane = threadIdx.x & 31;
    int before = 0;
    for (int64_t b0 = 0;; b0 += 32) {
        int const n = b0 + lane < a.B ? static_cast<int>((keys_of(a, b0 + lane) + KT - 1) / KT) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            int const y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        unsigned const past = __ballot_sync(0xffffffffu, before + upto > p);
        if (past != 0 || b0 + 32 >= a.B) {
            int const at = past != 0 ? __ffs(static_cast<int>(past)) - 1 : 31;
            first = before + __shfl_sync(0xffffffffu, upto - n, at);
            return b0 + at;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}

// SHARES: CTAs take even shares of all keys and leave parts of rows for
// merge_kernel; else a cluster of a.splits CTAs takes a KV head's keys and merges
// them itself.
template <int D, int R, int W, bool SHARES>
__global__ void __launch_bounds__(32 * W, Q8<D, R, W>::PER_SM) decode_q8_kernel(DecodeQ8Args a) {
    using C = Q8<D, R, W>;
    constexpr int MT = C::MT;
    extern __shared__ __align__(128) unsigned char smem[];
    uint4* sq = reinterpret_cast<uint4*>(smem + C::OFF_Q);
    float* sml = reinterpret_cast<float*>(smem + C::OFF_ML);
    float* sf = reinterpret_cast<float*>(smem + C::OFF_F);
    float* sx = reinterpret_cast<float*>(smem + C::OFF_X);
    int const tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    int const split = SHARES ? 0 : static_cast<int>(blockIdx.x) % a.splits;
    if (!SHARES && a.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // "this CTA runs"

    prior_kernels_done();

    int64_t b;            // sequence
    int unit, units = 0;  // KV head and row tile in it
    int at = 0, end = 0;  // SHARES: tiles still to do
    int t0 = 0, t1 = 0;
    bool first = true;
    if constexpr (SHARES) {
        units = static_cast<int>(a.Hkv * a.row_tiles);
        Shares const sh(tiles_before<C::KT>(a, a.B) * units, gridDim.x, W);
        at = sh.cut(blockIdx.x), end = sh.cut(blockIdx.x + 1);
        if (at >= end) return;
        int before;
        b = sequence_of<C::KT>(a, at / units, before);
        // the sequences before fill the first before * units tiles
        int const n = static_cast<int>((keys_of(a, b) + C::KT - 1) / C::KT), off = at - before * units;
        unit = off / n;
        t0 = off - unit * n;
    } else {
        uint32_t const all = blockIdx.x / a.splits, per = static_cast<uint32_t>(a.Hkv * a.row_tiles);
        b = all / per;
        unit = static_cast<int>(all % per);
    }
  for (;;) {
    int const kvh = unit / static_cast<int>(a.row_tiles);
    uint32_t const row0 = (unit - kvh * static_cast<int>(a.row_tiles)) * C::ROWS;  // first of the KV head's Tq * g query rows
    int const rows = static_cast<int>(min(static_cast<uint32_t>(a.Tq) * a.g - row0, uint32_t{C::ROWS}));
    int64_t const len = keys_of(a, b);

    // q's rows, loaded while the length is on its way
    constexpr int RPW = (C::ROWS + W - 1) / W, QV = (D + 127) / 128;  // rows of a warp, vectors of a lane
    float4 x[RPW][QV];
#pragma unroll
    for (int u = 0; u < RPW; ++u) {
        int const r = warp + u * W;
        uint32_t const row = row0 + r;
        int64_t const hq = static_cast<int64_t>(kvh) * a.g + row % a.g;
        bool const given = r < rows && hq < a.Hq;
        float const* q = a.q + b * a.q_b + (row / a.g) * a.q_t + hq * a.q_h;
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            int const d = 128 * i + 4 * lane;
            x[u][i] = given && d < D ? *reinterpret_cast<float4 const*>(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }

    // keys that row r of the tile sees; rows are ordered by token, then head
    auto visible = [&](int r) {
        int64_t const n = a.causal ? len - a.Tq + 1 + (row0 + r) / a.g : len;
        return static_cast<int>(max(int64_t{0}, n));
    };
    int const most = visible(rows - 1), least = visible(0);
    int const tiles = static_cast<int>(((SHARES ? len : most) + C::KT - 1) / C::KT);
    if constexpr (SHARES) {
        t1 = min(tiles, t0 + end - at);
    } else {
        t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / a.splits);
        t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / a.splits);
    }
    int const t1_seen = min(t1, (most + C::KT - 1) / C::KT);  // a row tile of earlier tokens sees fewer keys

    int8_t const* kb = a.k + b * a.k_b + kvh * a.k_h;
    int8_t const* vb = a.v + b * a.v_b + kvh * a.v_h;
    float const* ks = a.ks + b * a.ks_b + kvh * a.ks_h;
    float const* vs = a.vs + b * a.vs_b + kvh * a.vs_h;
    unsigned char* const ring = smem + C::RING * warp;
    uint32_t const ring_u = smem_u32(ring);
    // A tile of K or V into the ring: D / 16 lanes take a row. Keys past the last
    // one seen (of the range's last tile) read that one.
    auto fetch = [&](uint32_t dst, int8_t const* base, int64_t stride, int tile) {
        constexpr int LPR = D / 16, RPI = 32 / LPR;  // lanes per row, rows per instruction
        int const r0 = lane / LPR, c = lane % LPR, key = tile * C::KT;
        if (key + C::KT <= most && stride == D) {
            int8_t const* p = base + static_cast<int64_t>(key) * D + 16 * lane;
#pragma unroll
            for (int i = 0; i < C::KT / RPI; ++i) copy16(dst + C::place(r0 + i * RPI, c), p + 512 * i);
        } else if (key + C::KT <= most) {
            int8_t const* p = base + (key + r0) * stride + 16 * c;
#pragma unroll
            for (int i = 0; i < C::KT / RPI; ++i) copy16(dst + C::place(r0 + i * RPI, c), p + i * RPI * stride);
        } else {
#pragma unroll
            for (int i = 0; i < C::KT / RPI; ++i)
                copy16(dst + C::place(r0 + i * RPI, c), base + min(key + r0 + i * RPI, most - 1) * stride + 16 * c);
        }
    };
    float ksc[C::KV], vsc[C::KV];
    auto scales = [&](int tile) {
#pragma unroll
        for (int i = 0; i < C::KV; ++i) {
            int const j = min(tile * C::KT + 16 * i, most - 1) >> a.block_shift;
            ksc[i] = ks[j * a.ks_j];
            vsc[i] = vs[j * a.vs_j];
        }
    };
    int tile = t0 + warp;
    // groups: K, V of the first tile, K, V of the second
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (tile + u * W < t1_seen) fetch(ring_u + u * 2 * C::TILE, kb, a.k_t, tile + u * W);
        copies_close();
        if (tile + u * W < t1_seen) fetch(ring_u + (u * 2 + 1) * C::TILE, vb, a.v_t, tile + u * W);
        copies_close();
    }
    if (tile < t1_seen) scales(tile);

    // q's fragments and the factor of each row's scores.
#pragma unroll
    for (int u = 0; u < RPW; ++u) {
        int const r = warp + u * W;
        if (r >= C::ROWS) break;
        unsigned int top = 0;  // max |q| on the bit patterns: NaN above infinity above every number
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            top = max(max(top, __float_as_uint(x[u][i].x) & 0x7fffffffu), __float_as_uint(x[u][i].y) & 0x7fffffffu);
            top = max(max(top, __float_as_uint(x[u][i].z) & 0x7fffffffu), __float_as_uint(x[u][i].w) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        // the largest value into [2^29, 2^30): 2^(156 - e), e its biased exponent, where both factors are normal
        int const e = min(max(static_cast<int>(top >> 23), 31), 254);
        float const up = pow2_biased(283 - e), down = pow2_biased(e - 29);  // 2^(156 - e), 2^(e - 156)
        // NaN and infinity have no whole numbers: the whole row becomes NaN
        if (lane == 0) sf[r] = top >= 0x7f800000u ? __int_as_float(0x7fffffff) : down * (a.scale * kLog2e);
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            int const d = 128 * i + 4 * lane;
            if (d >= D) continue;
            // signed base-256 digits: a carry out of the lower bytes, then their signs
            auto digits = [&](float v) { return (static_cast<uint32_t>(__float2int_rn(v * up)) + 0x00808080u) ^ 0x00808080u; };
            uint32_t const n0 = digits(x[u][i].x), n1 = digits(x[u][i].y), n2 = digits(x[u][i].z), n3 = digits(x[u][i].w);
            uint32_t const lo01 = __byte_perm(n0, n1, 0x5140), hi01 = __byte_perm(n0, n1, 0x7362);
            uint32_t const lo23 = __byte_perm(n2, n3, 0x5140), hi23 = __byte_perm(n2, n3, 0x7362);
            // the lane and word of fragment that holds elements d .. d + 3
            int const c = d / 16, at = D == 64 ? c : (c % 8) / 2;
            int const word = 4 * (D == 64 ? 0 : 2 * (c / 8) + c % 2) + (d / 4) % 4, to = (r & 7) * 4 + at;
            uint2* f = reinterpret_cast<uint2*>(sq + ((r >> 3) * C::KS + word / 2) * (32 * C::QT) + to) + word % 2;
            uint32_t const d3 = __byte_perm(hi01, hi23, 0x7632), d2 = __byte_perm(hi01, hi23, 0x5410);
            uint32_t const d1 = __byte_perm(lo01, lo23, 0x7632), d0 = __byte_perm(lo01, lo23, 0x5410);
            if constexpr (R == 4) {  // rows g and g + 8 of the product: digits 3 and 1 for g < 4, 2 and 0 for g = 4 + row
                f[0] = make_uint2(d3, d1);
                f[32] = make_uint2(d2, d0);
            } else {  // digits 3 and 2 in one product, 1 and 0 in the next
                f[0] = make_uint2(d3, d2);
                f[64] = make_uint2(d1, d0);
            }
        }
    }
    __syncthreads();
    uint4 qf[C::QREG ? C::QT * MT * C::KS : 1];
    if constexpr (C::QREG) {
#pragma unroll
        for (int i = 0; i < C::QT * MT * C::KS; ++i) qf[i] = sq[i * 32 + lane];
    }
    float fac[MT];
    int seen[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        int const r = R == 4 ? g & 3 : 8 * m + g;
        fac[m] = sf[r];
        seen[m] = r < rows ? visible(r) : 0;
    }

    float lost[MT];              // units of the marked tiles, below
    float m_run[MT], l_run[MT];  // m_run: a whole number at or above the largest score, so that all factors are powers of two
    pair_t o[MT][D / 8];         // columns 2t and 2t + 1 of n-tile n
    constexpr int STRETCH = D == 64 ? 8 : 16;  // n-tiles of a lane's consecutive elements
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        m_run[m] = neg_inf(0.0f), l_run[m] = lost[m] = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[m][n] = pair(0.0f, 0.0f);
    }
    // scores of 8 MT rows and the KT keys of a tile in the ring
    auto scores_of = [&](unsigned char const* tk, float (&s)[MT][C::NK][2]) {
#pragma unroll
        for (int j = 0; j < C::NK; ++j) {
            uint32_t kr[C::KW];
#pragma unroll
            for (int i = 0; i < C::KW / 4; ++i) {
                uint4 const w = *reinterpret_cast<uint4 const*>(tk + C::place(8 * j + g, C::piece(i, t)));
                kr[4 * i] = w.x, kr[4 * i + 1] = w.y, kr[4 * i + 2] = w.z, kr[4 * i + 3] = w.w;
            }
            int hi[MT][4], lo[MT][4];
#pragma unroll
            for (int st = 0; st < C::KS; ++st) {
                uint32_t const b0 = kr[2 * st], b1 = kr[2 * st + 1];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    int const at = C::QT * (m * C::KS + st);
                    uint4 const qh = C::QREG ? qf[at] : sq[at * 32 + lane];
                    uint4 const ql = C::QREG ? qf[at + C::QT - 1] : sq[(at + C::QT - 1) * 32 + lane];
                    if (st == 0) {
                        mma_s8_first(hi[m], qh, b0, b1);
                        if constexpr (R > 4) mma_s8_first(lo[m], ql, b0, b1);
                    } else {
                        mma_s8(hi[m], qh, b0, b1);
                        if constexpr (R > 4) mma_s8(lo[m], ql, b0, b1);
                    }
                }
            }
            // digits' sums are below 2^22 each
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float const f = fac[m] * ksc[j / 2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (R == 4) {
                        float const x = fmaf(static_cast<float>(hi[m][e]), 65536.0f, static_cast<float>(hi[m][e + 2]));
                        float const y = __shfl_xor_sync(0xffffffffu, x, 16);
                        s[m][j][e] = (g < 4 ? fmaf(x, 256.0f, y) : fmaf(y, 256.0f, x)) * f;
                    } else {
                        s[m][j][e] = fmaf(static_cast<float>(hi[m][e] * 256 + hi[m][e + 2]), 65536.0f,
                                          static_cast<float>(lo[m][e] * 256 + lo[m][e + 2])) * f;
                    }
                }
            }
        }
    };
    auto mask = [&](int tile, float (&s)[MT][C::NK][2]) {
        if ((tile + 1) * C::KT <= least) return;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < C::NK; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (tile * C::KT + 8 * j + 2 * t + e >= seen[m]) s[m][j][e] = neg_inf(0.0f);
    };
    // V's scales relative to a power of two, whose biased exponent is returned: w < 2^14.
    // (R = 4: lanes g + 4 have the scores of lanes g; their rows of the product stay 0.)
    auto weights = [&](float (&w)[C::KV]) {
        unsigned top = 0;  // the largest |scale| on the bit patterns
#pragma unroll
        for (int i = 0; i < C::KV; ++i) top = max(top, __float_as_uint(vsc[i]) & 0x7fffffffu);
        int const e = min(max(static_cast<int>(top >> 23), 15), 253);
#pragma unroll
        for (int i = 0; i < C::KV; ++i) w[i] = R == 4 && g >= 4 ? 0.0f : vsc[i] * (pow2_biased(254 - e) * 8192.0f);
        return e;
    };
    // a row's largest score of a tile (four lanes share a row)
    auto largest = [&](float const (&s)[C::NK][2]) {
        float top = neg_inf(0.0f);
#pragma unroll
        for (int j = 0; j < C::NK; ++j) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        return fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    };
    // What a key adds to a row's output is its whole numbers times x = p vs, with p
    // relative to the whole number `local` next to the tile's largest score: x < 2^14.
    // Returns the lane's sum of p.
    auto terms = [&](float const (&s)[C::NK][2], float local, float const (&w)[C::KV], float (&x)[C::KV][4]) {
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < C::KV; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float const p0 = exp2_neg(s[2 * i + h][0] - local), p1 = exp2_neg(s[2 * i + h][1] - local);
                l += p0 + p1;
                float2 const v = unpair(mul2(pair(p0, p1), pair(w[i], w[i])));
                x[i][2 * h] = v.x, x[i][2 * h + 1] = v.y;
            }
        return l;
    };
    auto load_v = [&](unsigned char const* tv, uint32_t (&vr)[C::KV][4][C::VW]) {
#pragma unroll
        for (int i = 0; i < C::KV; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                int const r = 16 * i + 2 * t + (y & 1) + 8 * (y >> 1);
                if constexpr (D == 64) {
                    uint2 const w = *reinterpret_cast<uint2 const*>(tv + C::place(r, g >> 1) + 8 * (g & 1));
                    vr[i][y][0] = w.x, vr[i][y][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < C::VW / 4; ++c) {
                        uint4 const w = *reinterpret_cast<uint4 const*>(tv + C::place(r, 8 * c + g));
                        vr[i][y][4 * c] = w.x, vr[i][y][4 * c + 1] = w.y;
                        vr[i][y][4 * c + 2] = w.z, vr[i][y][4 * c + 3] = w.w;
                    }
                }
            }
    };
    // fragments of k16 steps: high parts in row g, low ones in row g + 8
    auto fragments = [&](float const (&x)[C::KV][4], uint32_t (&pa)[C::KV][4]) {
#pragma unroll
        for (int i = 0; i < C::KV; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) split2(x[i][2 * h], x[i][2 * h + 1], pa[i][2 * h], pa[i][2 * h + 1]);
    };
    // o += x V in units of `unit`, one word of V (four columns of lanes) at a time
    auto multiply = [&](uint32_t const (&pa)[MT][C::KV][4], float const (&unit)[MT], uint32_t const (&vr)[C::KV][4][C::VW]) {
#pragma unroll
        for (int w = 0; w < C::VW; ++w) {
            float c[MT][4][4];
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
                    for (int m = 0; m < MT; ++m) {
                        if (i == 0)
                            mma_f16_first(c[m][n], pa[m][i], b0, b1);
                        else
                            mma_f16(c[m][n], pa[m][i], b0, b1);
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    o[m][4 * w + n] = fma2(fma2(pair(c[m][n][2], c[m][n][3]), pair(kLowUnit, kLowUnit), pair(c[m][n][0], c[m][n][1])),
                                           pair(unit[m], unit[m]), o[m][4 * w + n]);
        }
    };
    // Tiles of the warp that are looked at again below: bit k % 32 of lane k / 32, the last
    // bit for all from there on.
    constexpr int kMarks = 1023;
    unsigned marks = 0;
    int k = 0;  // the warp's k-th tile
    for (int stage = 0; tile < t1_seen; tile += W, stage ^= 1, ++k) {
        unsigned char const* const tk = ring + stage * 2 * C::TILE;
        float s[MT][C::NK][2];
        copies_landed<3>();
        scores_of(tk, s);
        __syncwarp();  // the warp has read K; its place takes the tile after the next
        if (tile + 2 * W < t1_seen) fetch(ring_u + stage * 2 * C::TILE, kb, a.k_t, tile + 2 * W);
        copies_close();
        // the smallest score of each group of 16 keys, before the mask: keys past the end repeat the last one
        float low[MT][C::KV];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < C::KV; ++i)
                low[m][i] = fminf(fminf(s[m][2 * i][0], s[m][2 * i][1]), fminf(s[m][2 * i + 1][0], s[m][2 * i + 1][1]));
        mask(tile, s);
        unsigned vbad = 0;  // the largest |scale| of V's groups on the bit patterns
#pragma unroll
        for (int i = 0; i < C::KV; ++i) vbad = max(vbad, __float_as_uint(vsc[i]) & 0x7fffffffu);
        if (vbad >= 0x7f800000u) {  // NaN or infinity makes NaN of the rows that see its keys, and only of them
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int j = 0; j < C::NK; ++j)
                    if (fmaxf(s[m][j][0], s[m][j][1]) > neg_inf(0.0f)) l_run[m] += vsc[j / 2] * 0.0f;
#pragma unroll
            for (int i = 0; i < C::KV; ++i)
                if ((__float_as_uint(vsc[i]) & 0x7fffffffu) >= 0x7f800000u) vsc[i] = 0.0f;
        }
        float w[C::KV], reach[C::KV], unit[MT];  // reach: scores further than that from the largest have x < 2^-16
        int const ve = weights(w);
#pragma unroll
        for (int i = 0; i < C::KV; ++i)
            reach[i] = w[i] == 0.0f ? neg_inf(0.0f) : static_cast<float>(112 - static_cast<int>(__float_as_uint(fabsf(w[i])) >> 23));
        bool small = false;
        uint32_t pa[MT][C::KV][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float const top = largest(s[m]);
#pragma unroll
            for (int i = 0; i < C::KV; ++i) small |= low[m][i] < top + reach[i];
            float const m_new = fmaxf(m_run[m], ceilf(top));
            float const base = m_new == neg_inf(0.0f) ? 0.0f : m_new;
            if (__any_sync(0xffffffffu, m_new > m_run[m])) {
                float const alpha = exp2_neg(m_run[m] - base);
                l_run[m] *= alpha;
                lost[m] *= alpha;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) o[m][n] = mul2(o[m][n], pair(alpha, alpha));
                m_run[m] = m_new;
            }
            float const local = top == neg_inf(0.0f) ? base : ceilf(top), factor = exp2_neg(local - base);
            unit[m] = factor * pow2_biased(ve - 13);
            float x[C::KV][4];
            l_run[m] = fmaf(terms(s[m], local, w, x), factor, l_run[m]);
            fragments(x, pa[m]);
        }
        if (__any_sync(0xffffffffu, small)) {
            if (lane == min(k, kMarks) / 32) marks |= 1u << (min(k, kMarks) % 32);
#pragma unroll
            for (int m = 0; m < MT; ++m) lost[m] += unit[m];
        }
        if (tile + W < t1_seen) scales(tile + W);
        copies_landed<3>();
        uint32_t vr[C::KV][4][C::VW];
        load_v(tk + C::TILE, vr);
        __syncwarp();
        if (tile + 2 * W < t1_seen) fetch(ring_u + (stage * 2 + 1) * C::TILE, vb, a.v_t, tile + 2 * W);
        copies_close();
        multiply(pa, unit, vr);
    }
    copies_landed<0>();

    // Two fp16 parts hold x from 2^-16 on (2^-30 of the tile's largest) to 22 bits and lose up
    // to 2^-38 of what is smaller: of a marked tile, less than 2^-38 KT 128 units. Where that
    // may be more than 2^-22 of a sum (a column of V that is 0 at the keys of larger x), what the
    // marked tiles lost is added, in finer units.
    bool again = false;
    if (__any_sync(0xffffffffu, marks != 0)) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float const limit = lost[m] * (C::KT * 128.0f / 65536.0f);
            if (seen[m] == 0 || m_run[m] == neg_inf(0.0f) || (R == 4 && g >= 4)) continue;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
                float2 const y = unpair(o[m][n]);
                again |= fminf(fabsf(y.x), fabsf(y.y)) < limit;
            }
        }
    }
    if (__any_sync(0xffffffffu, again)) {
        int const count = k, first_tile = tile - k * W;
        auto marked = [&](int k) {  // the first marked tile from the k-th on, or `count`
            if (k >= kMarks) return __shfl_sync(0xffffffffu, marks, 31) >> 31 ? min(k, count) : count;
            unsigned const own = lane < k / 32 ? 0u : lane == k / 32 ? marks & ~0u << k % 32 : marks;
            unsigned const lanes = __ballot_sync(0xffffffffu, own != 0);
            int const from = __ffs(static_cast<int>(lanes)) - 1;
            unsigned const bits = __shfl_sync(0xffffffffu, own, max(from, 0));
            return lanes == 0 ? count : 32 * from + __ffs(static_cast<int>(bits)) - 1;
        };
        auto fetch_both = [&](int k, int stage) {
            if (k < count) {
                fetch(ring_u + stage * 2 * C::TILE, kb, a.k_t, first_tile + k * W);
                fetch(ring_u + (stage * 2 + 1) * C::TILE, vb, a.v_t, first_tile + k * W);
            }
            copies_close();
        };
        k = marked(0);
        fetch_both(k, 0);
#pragma unroll 1
        for (int stage = 0; k < count; stage ^= 1) {
            int const next = marked(k + 1);
            fetch_both(next, stage ^ 1);
            unsigned char const* const tk = ring + stage * 2 * C::TILE;
            float s[MT][C::NK][2], x[MT][C::KV][4], w[C::KV], unit[MT];
            tile = first_tile + k * W;
            scales(tile);
            copies_landed<1>();
            scores_of(tk, s);
            mask(tile, s);
#pragma unroll
            for (int i = 0; i < C::KV; ++i)
                if ((__float_as_uint(vsc[i]) & 0x7fffffffu) >= 0x7f800000u) vsc[i] = 0.0f;
            int const ve = weights(w);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float const top = largest(s[m]), base = m_run[m] == neg_inf(0.0f) ? 0.0f : m_run[m];
                float const local = top == neg_inf(0.0f) ? base : ceilf(top);
                unit[m] = exp2_neg(local - base) * pow2_biased(ve - 13);
                terms(s[m], local, w, x[m]);
            }
            uint32_t vr[C::KV][4][C::VW];
            load_v(tk + C::TILE, vr);
#pragma unroll 1
            for (bool more = true; more;) {  // three times at most: 2^-16 2^-51 2^-51 2^-51 < 2^-149
                more = false;
                uint32_t pa[MT][C::KV][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    unit[m] *= kFiner;
#pragma unroll
                    for (int i = 0; i < C::KV; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& y = x[m][i][e];
                            y = rest(y);
                            more |= y != 0.0f && fabsf(y) < kSmall;
                        }
                    fragments(x[m], pa[m]);
                }
                multiply(pa, unit, vr);
                more = __any_sync(0xffffffffu, more);
            }
            __syncwarp();  // the tile is read; its place takes another
            k = next;
        }
        copies_landed<0>();
    }

    // Warps to CTA: every warp's rows, maxima and sums. Columns 2t and 2t + 1 of
    // n-tile n are elements 32 t + n and 32 t + 16 + n of a 128-element stretch (D =
    // 64: 16 t + n and 16 t + 8 + n).
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        float l = l_run[m];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0 && (R > 4 || g < 4)) {
            sml[warp * C::ROWS + 8 * m + g] = m_run[m];
            sml[(W + warp) * C::ROWS + 8 * m + g] = l;
        }
        if (R > 4 || g < 4) {
            float* row = reinterpret_cast<float*>(ring) + (8 * m + g) * D;
#pragma unroll
            for (int n = 0; n < D / 8; n += 4) {
                float* p = row + (n / STRETCH) * 128 + 2 * STRETCH * t + n % STRETCH;
                float2 const v0 = unpair(o[m][n]), v1 = unpair(o[m][n + 1]), v2 = unpair(o[m][n + 2]),
                             v3 = unpair(o[m][n + 3]);
                *reinterpret_cast<float4*>(p) = make_float4(v0.x, v1.x, v2.x, v3.x);
                *reinterpret_cast<float4*>(p + STRETCH) = make_float4(v0.y, v1.y, v2.y, v3.y);
            }
        }
    }
    __syncthreads();
    // The CTA's sum of row r, elements 4 (i % (D / 4)) .., and the row's max and sum.
    auto weight = [](float m, float top) { return top == neg_inf(0.0f) ? 0.0f : exp2_neg(m - top); };
    auto add4 = [](float4& v, float w, float4 y) {
        v.x = fmaf(w, y.x, v.x);
        v.y = fmaf(w, y.y, v.y);
        v.z = fmaf(w, y.z, v.z);
        v.w = fmaf(w, y.w, v.w);
    };
    auto sum_warps = [&](int i, float& top, float& l) {
        int const r = i / (D / 4);
        top = neg_inf(0.0f), l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, sml[w * C::ROWS + r]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            float const f = weight(sml[w * C::ROWS + r], top);
            l = fmaf(f, sml[(W + w) * C::ROWS + r], l);
            add4(v, f, reinterpret_cast<float4 const*>(smem + C::RING * w)[i]);
        }
        return v;
    };
    auto store = [&](int i, float4 v, float l) {
        int const r = i / (D / 4), d = 4 * (i - r * (D / 4));
        uint32_t const row = row0 + r;
        int64_t const hq = static_cast<int64_t>(kvh) * a.g + row % a.g;
        if (hq >= a.Hq) return;
        float* p = a.out + b * a.o_b + (row / a.g) * a.o_t + hq * a.o_h + d * a.o_d;
        bool const none = l == 0.0f;  // no key seen; NaN goes through
        p[0] = none ? 0.0f : v.x / l;
        p[a.o_d] = none ? 0.0f : v.y / l;
        p[2 * a.o_d] = none ? 0.0f : v.z / l;
        p[3 * a.o_d] = none ? 0.0f : v.w / l;
    };
    int const items = rows * (D / 4);
    bool const whole = SHARES ? t0 == 0 && t1 == tiles : a.splits == 1;
    if (whole) {
        for (int i = tid; i < items; i += C::THREADS) {
            float top, l;
            float4 const v = sum_warps(i, top, l);
            store(i, v, l);
        }
    } else if constexpr (SHARES) {
        // a part of the rows: slot 0 if the share starts with it, else slot 1 (it ends the share)
        int64_t const slot = 2 * static_cast<int64_t>(blockIdx.x) + (first ? 0 : 1);
        float4* po = reinterpret_cast<float4*>(a.parts) + slot * (C::ROWS * D / 4);
        float* ps = a.parts + 2 * static_cast<int64_t>(gridDim.x) * (C::ROWS * D) + slot * (2 * C::ROWS);
        for (int i = tid; i < items; i += C::THREADS) {
            float top, l;
            po[i] = sum_warps(i, top, l);
            if (i % (D / 4) == 0) {
                ps[i / (D / 4)] = top;
                ps[C::ROWS + i / (D / 4)] = l;
            }
        }
    }
    if constexpr (SHARES) {
        at += t1 - t0;
        if (at >= end) return;
        first = false;
        t0 = 0;
        if (++unit == units) {
            unit = 0;
            do ++b;
            while (keys_of(a, b) == 0);  // `end` lies past a sequence that has keys
        }
        __syncthreads();  // the rings and statistics are read
        continue;
    }
    if (whole) return;
    // CTAs of the cluster: CTA s sums items [s * per, (s + 1) * per) of all of them.
    cg::cluster_group cluster = cg::this_cluster();
    int const per = (items + a.splits - 1) / a.splits;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA runs
    float4* recv = reinterpret_cast<float4*>(smem + C::OFF_R);           // [splits][per]
    for (int i = tid; i < items; i += C::THREADS) {
        float top, l;
        float4 const v = sum_warps(i, top, l);
        int const to = i / per, r = i / (D / 4);
        cluster.map_shared_rank(recv, to)[split * per + i - to * per] = v;
        // the row's statistics go with its first element and with every share's first
        if (i % (D / 4) == 0 || i == to * per) {
            float* px = cluster.map_shared_rank(sx, to) + split * 2 * C::ROWS + r;
            px[0] = top;
            px[C::ROWS] = l;
        }
    }
    cluster_sync();
    for (int i = split * per + tid; i < min(items, (split + 1) * per); i += C::THREADS) {
        int const r = i / (D / 4);
        float top = neg_inf(0.0f), l = 0.0f;
        for (int k = 0; k < a.splits; ++k) top = fmaxf(top, sx[k * 2 * C::ROWS + r]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < a.splits; ++k) {
            float const f = weight(sx[k * 2 * C::ROWS + r], top);
            l = fmaf(f, sx[k * 2 * C::ROWS + C::ROWS + r], l);
            add4(v, f, recv[k * per + i - split * per]);
        }
        store(i, v, l);
    }
    return;
  }
}

// The parts that the even shares left. A block takes `per_block` (1, 4 or 8) rows of
// a KV head's row tile; the kMergeWarps / per_block warps of a row share its parts.
constexpr int kMergeWarps = 16;
template <int D, int ROWS, int KT>
__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(DecodeQ8Args a, int G, int W, int per_block) {
    constexpr int LV = (D + 127) / 128;  // float4 of a row per lane
    __shared__ float4 sv[kMergeWarps][LV * 32];
    int const lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int const units = static_cast<int>(a.Hkv * a.row_tiles), wpr = kMergeWarps / per_block;
    int const r = blockIdx.y * per_block + warp / wpr, sub = warp % wpr;
    int64_t const b = blockIdx.x / static_cast<uint32_t>(units);
    int const u = static_cast<int>(blockIdx.x % static_cast<uint32_t>(units));
    // The lengths are read ahead of the wait: this grid starts when every block of the
    // shares' has ended, and each of those has waited for the kernels that wrote them.
    int const n = static_cast<int>((keys_of(a, b) + KT - 1) / KT);
    Shares const sh(tiles_before<KT>(a, a.B) * units, G, W);
    int const p0 = tiles_before<KT>(a, b) * units + u * n;
    int const c0 = n > 0 ? sh.owner(p0) : 0, c1 = n > 0 ? sh.owner(p0 + n - 1) : 0;
    // The shares are done and visible. Every block waits for that, those without work
    // too: this grid's end has to mean that the shares have ended.
    prior_kernels_done();
    if (n > 0 && c0 == c1) return;  // a whole unit: written by its CTA
    int const rt = static_cast<int>(a.row_tiles), kvh = u / rt;
    uint32_t const row = static_cast<uint32_t>((u - kvh * rt) * ROWS + r);
    int64_t const hq = static_cast<int64_t>(kvh) * a.g + row % a.g;
    bool const given = row < a.Tq * a.g && hq < a.Hq;
    int const parts = n > 0 ? c1 - c0 + 1 : 0;          // no keys: nobody's share, a row of zeros
    float const* stats = a.parts + 2 * G * (ROWS * D);
    // the first CTA may have come from the unit before, the others start with this one
    auto slot = [&](int k) { return static_cast<int64_t>(2 * (c0 + k) + (k == 0 && sh.cut(c0) < p0 ? 1 : 0)); };
    float top = neg_inf(0.0f), l = 0.0f;
    float4 v[LV];
#pragma unroll
    for (int i = 0; i < LV; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (given) {
        // Parts are loaded AT_ONCE at a time, the first ones together with the statistics.
        constexpr int AT_ONCE = 8 / LV, HELD = 4;
        float m[AT_ONCE];
        float4 y[AT_ONCE][LV];
        auto load = [&](int k0) {
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                int const k = k0 + u * wpr;
                int64_t const sl = slot(min(k, parts - 1));
                if (k < parts) {
                    m[u] = stats[sl * 2 * ROWS + r];
                    float4 const* po = reinterpret_cast<float4 const*>(a.parts) + (sl * ROWS + r) * (D / 4);
#pragma unroll
                    for (int i = 0; i < LV; ++i) y[u][i] = po[min(32 * i + lane, D / 4 - 1)];
                }
            }
        };
        if (sub < parts) load(sub);
        float pm[HELD], pl[HELD];  // of parts lane + 32 e
#pragma unroll
        for (int e = 0; e < HELD; ++e) {
            bool const in = lane + 32 * e < parts;
            float const* ps = stats + slot(in ? lane + 32 * e : 0) * 2 * ROWS + r;
            pm[e] = in ? ps[0] : neg_inf(0.0f);
            pl[e] = in ? ps[ROWS] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < HELD; ++e) top = fmaxf(top, pm[e]);
        for (int k = lane + 32 * HELD; k < parts; k += 32) top = fmaxf(top, stats[slot(k) * 2 * ROWS + r]);
        top = warp_max(top);
        auto weight = [&](float m) { return top == neg_inf(0.0f) ? 0.0f : exp2_neg(m - top); };
#pragma unroll
        for (int e = 0; e < HELD; ++e) l = fmaf(weight(pm[e]), pl[e], l);
        for (int k = lane + 32 * HELD; k < parts; k += 32) {
            float const* ps = stats + slot(k) * 2 * ROWS + r;
            l = fmaf(weight(ps[0]), ps[ROWS], l);
        }
        l = warp_sum(l);
        for (int k0 = sub; k0 < parts; k0 += AT_ONCE * wpr) {
            if (k0 != sub) load(k0);
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                if (k0 + u * wpr >= parts) break;
                float const w = weight(m[u]);
#pragma unroll
                for (int i = 0; i < LV; ++i) {
                    v[i].x = fmaf(w, y[u][i].x, v[i].x), v[i].y = fmaf(w, y[u][i].y, v[i].y);
                    v[i].z = fmaf(w, y[u][i].z, v[i].z), v[i].w = fmaf(w, y[u][i].w, v[i].w);
                }
            }
        }
    }
    if (wpr > 1) {
#pragma unroll
        for (int i = 0; i < LV; ++i) sv[warp][32 * i + lane] = v[i];
        __syncthreads();
        if (sub != 0) return;
        for (int k = 1; k < wpr; ++k)
#pragma unroll
            for (int i = 0; i < LV; ++i) {
                float4 const y = sv[warp + k][32 * i + lane];
                v[i].x += y.x, v[i].y += y.y, v[i].z += y.z, v[i].w += y.w;
            }
    }
    if (!given) return;
    float* out = a.out + b * a.o_b + (row / a.g) * a.o_t + hq * a.o_h;
    bool const none = l == 0.0f;
#pragma unroll
    for (int i = 0; i < LV; ++i) {
        if (32 * i + lane >= D / 4) continue;
        float* p = out + 4 * (32 * i + lane) * a.o_d;
        p[0] = none ? 0.0f : v[i].x / l;
        p[a.o_d] = none ? 0.0f : v[i].y / l;
        p[2 * a.o_d] = none ? 0.0f : v[i].z / l;
        p[3 * a.o_d] = none ? 0.0f : v[i].w / l;
    }
}

// Scratch for the parts, in stream order, from a pool of the library's own for
// each device: the default pool would give the memory back to the driver at
// every synchronisation.
int scratch_alloc(void** p, size_t bytes, cudaStream_t stream) {
    static std::mutex mu;
    static std::map<int, cudaMemPool_t> pools;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8: no CUDA device.");
    cudaMemPool_t pool = nullptr;
    {
        std::lock_guard<std::mutex> lock(mu);
        auto const it = pools.find(dev);
        if (it != pools.end()) {
            pool = it->second;
        } else {
            // the first call of all may be one that is captured: making a pool is no work on its stream
            cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
            cudaThreadExchangeStreamCaptureMode(&mode);
            cudaMemPoolProps props{};
            props.allocType = cudaMemAllocationTypePinned;
            props.location.type = cudaMemLocationTypeDevice;
            props.location.id = dev;
            cudaError_t e = cudaMemPoolCreate(&pool, &props);
            uint64_t keep = UINT64_MAX;
            if (e == cudaSuccess) e = cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep);
            cudaThreadExchangeStreamCaptureMode(&mode);
            if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8 scratch: %s", cudaGetErrorString(e));
            pools[dev] = pool;
        }
    }
    cudaError_t const e = cudaMallocFromPoolAsync(p, bytes, pool, stream);
    if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8 scratch: %s", cudaGetErrorString(e));
    return ANN_OK;
}

// Kernel attributes, once per device.
template <typename K>
int prepare(K kernel, size_t smem, bool wide_cluster, std::set<int>& ready, std::mutex& mu) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8: no CUDA device.");
    std::lock_guard<std::mutex> lock(mu);
    if (ready.count(dev) != 0) return ANN_OK;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e == cudaSuccess && wide_cluster)
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8 setup: %s", cudaGetErrorString(e));
    ready.insert(dev);
    return ANN_OK;
}

// One launch, a cluster of CTAs per KV head: for calls of little work.
template <int D, int R>
struct Clusters {
    static constexpr int W = 4;
    using C = Q8<D, R, W>;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attrs[2] = {{}, overlapping()};

    explicit Clusters(int splits) {
        cudaLaunchAttribute& attr = attrs[0];
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = static_cast<unsigned>(splits);
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.gridDim = dim3(static_cast<unsigned>(splits));
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.attrs = attrs;
        cfg.numAttrs = 2;
    }
    Clusters(Clusters const&) = delete;

    // Clusters of 1 .. kMaxCluster CTAs that the device holds at once.
    static int room(const std::array<int, kMaxCluster + 1>*& out) {
        static std::mutex mu;
        static std::set<int> ready;
        static std::map<int, std::array<int, kMaxCluster + 1>> rooms;
        auto const kernel = decode_q8_kernel<D, R, W, false>;
        ANN_TRY(prepare(kernel, C::SMEM, true, ready, mu));
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8: no CUDA device.");
        std::lock_guard<std::mutex> lock(mu);
        auto it = rooms.find(dev);
        if (it == rooms.end()) {
            std::array<int, kMaxCluster + 1> r{};
            for (int s = 1; s <= kMaxCluster; ++s) {
                Clusters of(s);
                cudaError_t const e = cudaOccupancyMaxActiveClusters(&r[s], kernel, &of.cfg);
                if (e != cudaSuccess) return fail(ANN_ECUDA, "attentionDecodeQ8 setup: %s", cudaGetErrorString(e));
            }
            it = rooms.emplace(dev, r).first;
        }
        out = &it->second;
        return ANN_OK;
    }
    int launch(ann_stream stream, const DecodeQ8Args& a, int64_t units) {
        if (units * a.splits > INT32_MAX) return fail(ANN_ENOTSUP, "attentionDecodeQ8: grid too large.");
        cfg.gridDim = dim3(static_cast<unsigned>(units * a.splits));
        cfg.stream = as_stream(stream);
        cudaLaunchKernelEx(&cfg, decode_q8_kernel<D, R, W, false>, a);
        return check_launch("attentionDecodeQ8");
    }
};

// Even shares of all keys for as many CTAs as fit the GPU, then the merge of the
// rows that several CTAs share.
template <int D, int R>
int launch_shares(ann_stream stream, DecodeQ8Args& a, int64_t units) {
    constexpr int W = 4;
    using C = Q8<D, R, W>;
    auto const kernel = decode_q8_kernel<D, R, W, true>;
    static std::mutex mu;
    static std::set<int> ready;
    ANN_TRY(prepare(kernel, C::SMEM, false, ready, mu));
    int64_t const G = std::min<int64_t>(kMaxShares, int64_t{sm_count()} * C::PER_SM);
    void* parts = nullptr;
    ANN_TRY(scratch_alloc(&parts, sizeof(float) * 2 * G * (C::ROWS * D + 2 * C::ROWS), as_stream(stream)));
    a.parts = static_cast<float*>(parts);
    launch_overlapping(kernel, dim3(static_cast<unsigned>(G)), C::THREADS, C::SMEM, as_stream(stream), a);
    int rc = check_launch("attentionDecodeQ8");
    if (rc == ANN_OK) {
        // Few units have many parts each, so all warps of a block go to one row; many fill the
        // GPU with a warp or two a row (rows a block of 1 / 4 / 8, us of both kernels: 4 units, 1 x
        // 131072 keys, 37.4 / 40.8 / 44.5; 32, 4 x 65536, 101 / 97 / 97; 64, 8 x 32768, 107 / 97 / 96).
        int const rows = static_cast<int>(std::min<int64_t>(C::ROWS, a.Tq * a.g)), per_block = units < G / 8 ? 1 : std::min(8, C::ROWS);
        dim3 const grid(static_cast<unsigned>(units), static_cast<unsigned>(ceil_div(rows, per_block)));
        launch_overlapping(merge_kernel<D, C::ROWS, C::KT>, grid, 32 * kMergeWarps, 0, as_stream(stream), a,
                           static_cast<int>(G), W, per_block);
        rc = check_launch("attentionDecodeQ8");
    }
    cudaFreeAsync(parts, as_stream(stream));
    return rc;
}

// Which way, and how many splits: the least of these costs, in tiles' times of a
// warp on a full SM (2.2 us for 8 KB: 12 warps share an SM's part of HBM).
//  * Clusters of S: rounds of as many as the device holds at once (of six CTAs, two an
//    SM, 45 and not 49), each ceil(tiles / 4 S) tiles a warp and about
//    one tile's time to start and to merge. A tile takes less where the grid
//    does not fill the GPU, though not in proportion, and no less than 0.45.
//  * Even shares: their tiles a warp, and about 1.5 tiles' times for the second
//    launch and for each part of a KV head that a CTA meets.
// Measured (us, clusters at their best S / shares): 8 x 2048 keys, 32 KV heads 28 /
// 38; 12 x 4096 keys of 64, 4 heads, four tokens 13 / 17; 31 x 7345 keys of 64, 6
// heads 41 / 47; 16 x 32768 keys, 8 heads 176 / 174; 1 x 131072 keys, 4 heads 69 / 38.
template <int D, int R>
struct Plan {
    using C = Q8<D, R, 4>;
    int64_t row_tiles = 0, units = 0;
    int splits = 0;      // 0: even shares
    double cost = 1e300;

    int make(const DecodeQ8Args& a) {
        row_tiles = ceil_div(a.Tq * a.g, C::ROWS);
        units = a.B * a.Hkv * row_tiles;
        int64_t const tiles = ceil_div(a.cap, C::KT);
        if (units > INT32_MAX) return fail(ANN_ENOTSUP, "attentionDecodeQ8: grid too large.");
        double const slots = static_cast<double>(sm_count()) * C::PER_SM, all = static_cast<double>(units) * tiles;
        const std::array<int, kMaxCluster + 1>* room = nullptr;
        ANN_TRY((Clusters<D, R>::room(room)));
        for (int s = 1; s <= kMaxCluster && (s == 1 || (s - 1) * 4 < tiles); ++s) {
            if ((*room)[s] == 0) continue;
            double const full = std::min(1.0, static_cast<double>(units) * s / slots);
            double const c = std::ceil(static_cast<double>(units) / (*room)[s]) *
                             (std::ceil(tiles / (4.0 * s)) * std::max(0.45, 0.3 + 0.7 * full) + 1.0);
            if (c < cost) cost = c, splits = s;
        }
        // the shares' tiles are counted in 32 bits
        double const shares = all > INT32_MAX / 2 ? 1e300 : all / (4.0 * slots) + 1.5 * (2.0 + static_cast<double>(units) / slots);
        if (shares < cost) cost = shares, splits = 0;
        return ANN_OK;
    }
    int launch(ann_stream stream, DecodeQ8Args& a) const {
        a.row_tiles = row_tiles;
        a.splits = std::max(1, splits);
        return splits > 0 ? Clusters<D, R>(splits).launch(stream, a, units) : launch_shares<D, R>(stream, a, units);
    }
};

template <int D, int R>
int launch(ann_stream stream, DecodeQ8Args& a) {
    Plan<D, R> plan;
    ANN_TRY(plan.make(a));
    return plan.launch(stream, a);
}

// Query rows of a CTA. Sixteen read the cache half as often as eight, but a tile takes
// a warp 1.1 times as long, the start and the end one microsecond (0.6 tiles) more, and
// their registers leave 8 warps an SM instead of 12 (16 x 16384 keys of 64, 8 heads of
// sixteen rows: 95 us against 113; 12 x 4096, 4 heads: 15.0 against 12.8; 1 x 300, 3
// heads: 8.2 against 6.2). Heads of 256 take eight: sixteen rows' sums and fragments do
// not fit the registers (2 x 65536 keys, 2 heads of sixteen rows: 81 us against 57; 16 x
// 8192, 4 heads: 134 against 94).
template <int D>
int launch_rows(ann_stream stream, DecodeQ8Args& a) {
    if (a.Tq > INT32_MAX / 2 / int64_t{a.g}) return fail(ANN_ENOTSUP, "attentionDecodeQ8: more than 2^30 rows.");
    int64_t const rows = a.Tq * a.g;
    if constexpr (D <= 128) {
        if (rows <= 4) return launch<D, 4>(stream, a);
        if (rows > 8) {
            Plan<D, 8> eight;
            Plan<D, 16> sixteen;
            ANN_TRY(eight.make(a));
            ANN_TRY(sixteen.make(a));
            if (1.1 * sixteen.cost + 0.6 <= eight.cost) return sixteen.launch(stream, a);
            return eight.launch(stream, a);
        }
    }
    return launch<D, 8>(stream, a);
}

int decode_q8(ann_stream stream, const ann_view* q_v, const ann_view* k_v, const ann_view* v_v, const ann_view* ks_v,
              const ann_view* vs_v, const ann_view* len_v, const ann_view* o_v, float scale, uint32_t g, uint32_t block,
              int layout, int causal) {
    if (g == 0u) return fail(ANN_EINVAL, "attentionDecodeQ8 requires queriesPerKvGroup > 0.");
    if (layout != ANN_LAYOUT_BTHD && layout != ANN_LAYOUT_BHTD)
        return fail(ANN_EINVAL, "attentionDecodeQ8: invalid kv layout.");
    if (block == 0u) return fail(ANN_EINVAL, "attentionDecodeQ8 requires tokensPerScale > 0.");
    Dims q, k, v, ks, vs, o;
    ANN_TRY(to_dims_flat(q_v, sizeof(float), "attentionDecodeQ8 Q", q));
    ANN_TRY(to_dims_flat(k_v, 1, "attentionDecodeQ8 K", k));
    ANN_TRY(to_dims_flat(v_v, 1, "attentionDecodeQ8 V", v));
    ANN_TRY(to_dims_flat(ks_v, sizeof(float), "attentionDecodeQ8 K scales", ks));
    ANN_TRY(to_dims_flat(vs_v, sizeof(float), "attentionDecodeQ8 V scales", vs));
    ANN_TRY(to_dims_flat(o_v, sizeof(float), "attentionDecodeQ8 out", o));
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
        ANN_TRY(to_dims_flat(len_v, sizeof(int32_t), "attentionDecodeQ8 lengths", len));
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
    g = static_cast<uint32_t>(std::min<int64_t>(g, Hq));  // a larger group holds no more queries
    a.Hkv = ceil_div(Hq, int64_t{g});  // KV heads that queries read
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
