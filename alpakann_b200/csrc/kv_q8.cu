// kv_q8.cu -- a KV cache held in 8 bits: append and read-back.
//
// A cache value is a whole number n in [-127, 127]; it stands for n * s, with
// one fp32 scale s per KV head and block of `block` tokens:
//   k_cache, v_cache int8 [B, Hkv, Tcap, D] (or BTHD), scales [B, Hkv, ceil(Tcap / block)].
//
// append: s' = max(|s| of the block's earlier rows, max|x| times fp32's 1/127 over
// the new rows in the block); a new value becomes the whole number nearest to the exact
// quotient x / s' (ties to even); where s' grew, or s was negative, the block's earlier
// values are rounded anew from n * s / s'. The rounding is exact, not that of a 32-bit
// quotient, so any implementation of this definition gives the same integers.
// A NaN or infinity in a new row makes its block's scale NaN or infinite, so
// the block reads back as NaN / infinity instead of as wrong finite values.
//
// Both are bound by HBM: append reads 4 bytes and writes 1 per value, the
// read-back reads 1 and writes 4. Measured at 4 x 2048 tokens, 8 heads of 128: append
// 24 us (0.54 of the bytes' time at the copy rate: the block's largest value has to be
// known before the first is written, so loads and stores alternate), read-back 23 us (0.84
// of the bytes of 4 x 3048 tokens); one token of 8 sequences 2.5 and 4.0 us, a launch each.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "overlap.cuh"
#include "reduce.cuh"

namespace ann {
namespace {

__device__ unsigned int g_kv_q8_error;

constexpr int kThreads = 256;
constexpr int kHeld = 8;  // 16-byte vectors of a thread kept between append's two passes

struct CacheTensor {
    int8_t* q;
    float* scale;
    int64_t q_b, q_h, q_t, q_d;  // element strides
    int64_t s_b, s_h, s_j;
};

struct AppendArgs {
    CacheTensor c[2];
    const float* x[2];
    int64_t x_b[2], x_t[2], x_h[2], x_d[2];
    const int32_t* pos;
    const int32_t* counts;  // may be null: every row
    int64_t pos_s, counts_s;
    int64_t Tn, D, cap, block;
    FastDiv touched, heads;  // blocks a sequence's rows can reach, KV heads
    FastDiv blocks;          // by a block's tokens
    FastDiv row;             // by the items of a row: 4 aligned values (vec) or one
    int rows;                // whole rows of one item a thread (STEP)
    int vec;
};

// The whole number nearest to x / s, exactly, ties to even; |x| <= 127 s up to
// the roundings of s. t is within 2^-16 of the quotient, so rint(t) is off by one
// at most; r = x - n s is exact in 32 bits (a multiple of half an ulp of s, at
// most 2^24 of them), and comparing it with s / 2 puts n right.
__device__ __forceinline__ int nearest(float x, float s, float inv) {
    float n = rintf(x * inv);
    float const r = fmaf(-n, s, x), half = 0.5f * s;
    bool const odd = static_cast<int>(n) & 1;
    if (r > half || (r == half && odd)) n += 1.0f;
    if (r < -half || (r == -half && odd)) n -= 1.0f;
    return max(-127, min(127, static_cast<int>(n)));
}
// Four of them as bytes. Adding 1.5 * 2^23 rounds x / s to a whole number whose low
// byte is the sum's; where it may be off, the remainder says so, and the value
// (one in thousands) is rounded as above.
__device__ __forceinline__ uint32_t nearest4(float4 x, float s, float inv) {
    float const magic = 12582912.0f;
    float const y0 = fmaf(x.x, inv, magic), y1 = fmaf(x.y, inv, magic), y2 = fmaf(x.z, inv, magic),
                y3 = fmaf(x.w, inv, magic);
    float const r0 = fmaf(magic - y0, s, x.x), r1 = fmaf(magic - y1, s, x.y), r2 = fmaf(magic - y2, s, x.z),
                r3 = fmaf(magic - y3, s, x.w);
    uint32_t const lo = __byte_perm(__float_as_uint(y0), __float_as_uint(y1), 0x0040),
                   hi = __byte_perm(__float_as_uint(y2), __float_as_uint(y3), 0x0040);
    uint32_t bytes = __byte_perm(lo, hi, 0x5410);
    if (fmaxf(fmaxf(fabsf(r0), fabsf(r1)), fmaxf(fabsf(r2), fabsf(r3))) >= 0.5f * s) {
        char4 const n = make_char4(nearest(x.x, s, inv), nearest(x.y, s, inv), nearest(x.z, s, inv), nearest(x.w, s, inv));
        bytes = *reinterpret_cast<uint32_t const*>(&n);
    }
    return bytes;
}
// The larger of |x| and m, NaN if either is.
__device__ __forceinline__ float max_abs(float x, float m) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(fabsf(x)), "f"(m));
    return v;
}
// The same in 64 bits, for scales so small that the 32-bit remainder is not
// exact, and for requantised values n_old * s_old / s.
__device__ __forceinline__ int nearest64(double x, double s) {
    return static_cast<int>(fmin(fmax(rint(x / s), -127.0), 127.0));
}

// TH threads. STEP: a row's items divide them, and they step over rows.
template <bool STEP, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) append_kernel(AppendArgs const __grid_constant__ a) {
    __shared__ unsigned int red[TH / 32];
    uint32_t const bhk = a.touched.div(blockIdx.x), jb = blockIdx.x - bhk * a.touched.d;
    int const kv = static_cast<int>(bhk & 1u);
    uint32_t const ub = a.heads.div(bhk >> 1);
    int64_t const b = ub, h = (bhk >> 1) - ub * a.heads.d;

    prior_kernels_done();
    int64_t const start = a.pos[b * a.pos_s];
    int64_t count = a.Tn;
    if (a.counts != nullptr) count = min(a.Tn, max(int64_t{0}, static_cast<int64_t>(a.counts[b * a.counts_s])));
    int64_t const first = max(start, int64_t{0}), end = min(start + count, a.cap);
    if (threadIdx.x == 0 && count > 0 && (start < 0 || start + count > a.cap))
        atomicOr(&g_kv_q8_error, ANN_DEVERR_CACHE_RANGE);
    int64_t const j = a.blocks.div(static_cast<uint32_t>(min(first, a.cap))) + jb;
    int64_t const lo = max(first, j * a.block), hi = min(end, (j + 1) * a.block);
    if (lo >= hi) return;

    CacheTensor const& c = a.c[kv];
    float const* x = a.x[kv] + b * a.x_b[kv] + h * a.x_h[kv];
    int64_t const x_t = a.x_t[kv], x_d = a.x_d[kv];
    x += (lo - start) * x_t;
    int8_t* q = c.q + b * c.q_b + h * c.q_h;
    float* scale = c.scale + b * c.s_b + h * c.s_h + j * c.s_j;
    int const rows = static_cast<int>(hi - lo), D = static_cast<int>(a.D);

    // The first kHeld items of a thread stay in registers between the two passes,
    // loaded at once; later ones are read again, from L2. (Four held and five blocks an
    // SM: 27 us, eight and four 24, at 4 x 2048 tokens in blocks of 64.)
    int const per = static_cast<int>(a.row.d), items = rows * per;  // of a row, of the new rows
    int const r0 = static_cast<int>(a.row.div(threadIdx.x)), c0 = static_cast<int>(threadIdx.x) - r0 * per;
    auto place = [&](int u, int& r, int& col) {  // item threadIdx.x + u * TH
        if constexpr (STEP) {
            r = r0 + u * a.rows;
            col = c0;
        } else {
            int const i = static_cast<int>(threadIdx.x) + u * TH;
            r = static_cast<int>(a.row.div(i));
            col = i - r * per;
        }
    };
    int const mine = (items - static_cast<int>(threadIdx.x) + TH - 1) / TH;  // items of this thread
    int64_t const x_u = STEP ? a.rows * x_t : 0, q_u = STEP ? a.rows * c.q_t : 0;
    float const* const x0 = x + r0 * x_t + 4 * c0;
    int8_t* const q0 = q + (lo + r0) * c.q_t + 4 * c0;
    auto vector = [&](int u) {
        if constexpr (STEP) return *reinterpret_cast<float4 const*>(x0 + u * x_u);
        int r, col;
        place(u, r, col);
        return *reinterpret_cast<float4 const*>(x + r * x_t + 4 * col);
    };
    float most = 0.0f;
    auto raise = [&](float4 v) { most = max_abs(v.x, max_abs(v.y, max_abs(v.z, max_abs(v.w, most)))); };
    float4 held[kHeld];
    if (a.vec) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u) held[u] = u < mine ? vector(u) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < kHeld; ++u) raise(held[u]);
        if constexpr (STEP) {
            float const* p = x0 + kHeld * x_u;
#pragma unroll 4
            for (int u = kHeld; u < mine; ++u, p += x_u) raise(*reinterpret_cast<float4 const*>(p));
        } else {
            for (int u = kHeld; u < mine; ++u) raise(vector(u));
        }
    } else {
        for (int u = 0; u < mine; ++u) {
            int r, col;
            place(u, r, col);
            most = max_abs(x[r * x_t + col * x_d], most);
        }
    }
    // on the bit patterns: ordered like the values, infinity above every number and NaN above infinity
    unsigned int top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    bool const begun = j * a.block < lo;  // the block holds earlier rows
    float const stored = begun ? *scale : 0.0f, old = fabsf(stored);  // a caller may have stored a negative one
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TH / 32; ++w) top = max(top, red[w]);
    unsigned int const want = __float_as_uint(__uint_as_float(top) * (1.0f / 127.0f));
    float const s = __uint_as_float(max(want, __float_as_uint(old)));
    if (threadIdx.x == 0) *scale = s;  // every thread has read the old one before the barrier above

    bool const finite = __float_as_uint(s) < 0x7f800000u && s > 0.0f;
    if (begun && __float_as_uint(s) != __float_as_uint(stored)) {
        int64_t const t0 = j * a.block;
        int const early = static_cast<int>(lo - t0);
        for (int i = threadIdx.x; i < early * D; i += TH) {
            int const r = i / D, d = i - r * D;
            int8_t* p = q + (t0 + r) * c.q_t + d * c.q_d;
            *p = static_cast<int8_t>(finite ? nearest64(static_cast<double>(*p) * stored, s) : 0);
        }
    }
    // 64-bit rounding for tiny scales: the remainder's ulp argument needs normal numbers
    bool const usual = finite && s >= 1e-30f;
    float const inv = 1.0f / s;
    auto round1 = [&](float v) { return usual ? nearest(v, s, inv) : finite ? nearest64(v, s) : 0; };
    auto four = [&](float4 v) {
        uint32_t bytes;
        if (usual) {
            bytes = nearest4(v, s, inv);
        } else {
            char4 const n = make_char4(round1(v.x), round1(v.y), round1(v.z), round1(v.w));
            bytes = *reinterpret_cast<uint32_t const*>(&n);
        }
        return bytes;
    };
    auto write4 = [&](int u, float4 v) {
        int r, col;
        place(u, r, col);
        *reinterpret_cast<uint32_t*>(STEP ? q0 + u * q_u : q + (lo + r) * c.q_t + 4 * col) = four(v);
    };
    if (a.vec) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (u < mine) write4(u, held[u]);
        if constexpr (STEP) {
            float const* p = x0 + kHeld * x_u;
            int8_t* to = q0 + kHeld * q_u;
#pragma unroll 2
            for (int u = kHeld; u < mine; ++u, p += x_u, to += q_u)
                *reinterpret_cast<uint32_t*>(to) = four(*reinterpret_cast<float4 const*>(p));
        } else {
            for (int u = kHeld; u < mine; ++u) write4(u, vector(u));
        }
    } else {
        for (int u = 0; u < mine; ++u) {
            int r, col;
            place(u, r, col);
            q[(lo + r) * c.q_t + col * c.q_d] = static_cast<int8_t>(round1(x[r * x_t + col * x_d]));
        }
    }
}

struct ReadArgs {
    CacheTensor c[2];
    float* out[2];
    int64_t o_b[2], o_h[2], o_t[2], o_d[2];
    const int32_t* lengths;  // may be null: every row
    int64_t len_s;
    int64_t D, Tout;
    FastDiv chunks, heads;  // chunks of a thread block's items per (batch, head), KV heads
    FastDiv row, block;     // by the items of a row (4 aligned values, or one), by a block's tokens
    uint32_t rows;          // whole rows of one item a thread (STEP)
    int vec;
};


// Items of a thread whose loads go out together (eight: 23.0 us for 22.8 below), ahead of the
// stores of those before (load_input; ordinary loads: 24.4).
constexpr int kReadAtOnce = 4;

// Signed byte `at` of w as fp32: its bits with the sign flipped, 128 + n, are the low
// ones of 2^23 + 128 + n.
__device__ __forceinline__ float byte_of(uint32_t w, uint32_t at) {
    return __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7650 | at)) - 8388736.0f;
}

// A thread takes EACH items, which share what it computes of its place.
template <bool VEC, bool STEP, int EACH>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadArgs const __grid_constant__ a) {
    uint32_t const bhk = a.chunks.div(blockIdx.x), chunk = blockIdx.x - bhk * a.chunks.d;
    int const kv = static_cast<int>(bhk & 1u);
    uint32_t const ub = a.heads.div(bhk >> 1);
    int64_t const b = ub, h = (bhk >> 1) - ub * a.heads.d;
    CacheTensor const& c = a.c[kv];
    int8_t const* q = c.q + b * c.q_b + h * c.q_h;
    float const* scale = c.scale + b * c.s_b + h * c.s_h;
    float* out = a.out[kv] + b * a.o_b[kv] + h * a.o_h[kv];
    int64_t const o_t = a.o_t[kv], o_d = a.o_d[kv];
    uint32_t const per = a.row.d, base = chunk * (kThreads * EACH) + threadIdx.x;
    uint32_t t = a.row.div(base), col = base - t * per;
    uint32_t const all = static_cast<uint32_t>(a.Tout);
    int64_t const q_u = STEP ? a.rows * c.q_t : 0, o_u = STEP ? a.rows * o_t : 0;
    int8_t const* p = q + t * c.q_t + (VEC ? 4 * col : col * c.q_d);
    float* o = out + t * o_t + (VEC ? 4 * col : col * o_d);
    prior_kernels_done();
    // The length is on its way with the first loads: rows past it are read (they are
    // part of the cache) and not written.
    uint32_t const length = a.lengths != nullptr ? static_cast<uint32_t>(max(0, a.lengths[b * a.len_s])) : all;
#pragma unroll 1
    for (int u0 = 0; u0 < EACH && t < all; u0 += kReadAtOnce) {
        float s[kReadAtOnce];
        uint32_t n[kReadAtOnce];
        uint32_t const t0 = t;
#pragma unroll
        for (int u = 0; u < kReadAtOnce; ++u) {
            bool const in = t < all;
            s[u] = in ? load_input(scale + a.block.div(t) * c.s_j) : 0.0f;
            if constexpr (VEC)
                n[u] = in ? load_input(reinterpret_cast<uint32_t const*>(p)) : 0u;
            else
                n[u] = in ? static_cast<uint32_t>(static_cast<int>(*p)) : 0u;
            if constexpr (STEP) {
                t += a.rows, p += q_u;
            } else {
                uint32_t const i = base + (u0 + u + 1) * kThreads;
                t = a.row.div(i), col = i - t * per;
                p = q + t * c.q_t + (VEC ? 4 * col : col * c.q_d);
            }
        }
        uint32_t const rows = min(all, length);
        uint32_t tu = t0;
#pragma unroll
        for (int u = 0; u < kReadAtOnce; ++u) {
            if constexpr (!STEP) {
                uint32_t const i = base + (u0 + u) * kThreads;
                tu = a.row.div(i), col = i - tu * per;
                o = out + tu * o_t + (VEC ? 4 * col : col * o_d);
            }
            if (tu < rows) {
                if constexpr (VEC)
                    *reinterpret_cast<float4*>(o) = make_float4(byte_of(n[u], 0) * s[u], byte_of(n[u], 1) * s[u],
                                                                byte_of(n[u], 2) * s[u], byte_of(n[u], 3) * s[u]);
                else
                    *o = static_cast<float>(static_cast<int>(n[u])) * s[u];
            }
            if constexpr (STEP) tu += a.rows, o += o_u;
        }
    }
}

// The two caches and their scales, checked against each other.
int cache_tensors(const char* what, const ann_view* const qv[2], const ann_view* const sv[2], uint32_t block, int layout,
                  Dims q[2], Dims s[2]) {
    if (layout != ANN_LAYOUT_BTHD && layout != ANN_LAYOUT_BHTD) return fail(ANN_EINVAL, "%s: invalid kv layout.", what);
    if (block == 0) return fail(ANN_EINVAL, "%s requires tokensPerScale > 0.", what);
    for (int k = 0; k < 2; ++k) {
        ANN_TRY(to_dims_flat(qv[k], 1, what, q[k]));
        ANN_TRY(to_dims_flat(sv[k], sizeof(float), what, s[k]));
    }
    if (q[0].rank != 4 || q[1].rank != 4) return fail(ANN_EINVAL, "%s expects rank-4 caches.", what);
    if (!same_extents(q[0], q[1])) return fail(ANN_EINVAL, "%s: K and V cache extents differ.", what);
    int const tok = layout == ANN_LAYOUT_BTHD ? 1 : 2, head = 3 - tok;
    for (int k = 0; k < 2; ++k)
        if (s[k].rank != 3 || s[k].ext[0] != q[k].ext[0] || s[k].ext[1] != q[k].ext[head] ||
            s[k].ext[2] != ceil_div(q[k].ext[tok], block))
            return fail(ANN_EINVAL, "%s: scales %s do not match the cache %s with %u tokens a scale.", what,
                        extents_str(s[k]).c_str(), extents_str(q[k]).c_str(), block);
    return ANN_OK;
}

CacheTensor tensor_of(const Dims& q, const Dims& s, int layout) {
    int const tok = layout == ANN_LAYOUT_BTHD ? 1 : 2, head = 3 - tok;
    return CacheTensor{static_cast<int8_t*>(q.data), static_cast<float*>(s.data), q.str[0], q.str[head], q.str[tok],
                       q.str[3], s.str[0], s.str[1], s.str[2]};
}

// A rank-1 int32 view with one entry per sequence.
int per_sequence(const ann_view* v, const char* what, int64_t B, const int32_t*& p, int64_t& stride) {
    Dims d;
    ANN_TRY(to_dims_flat(v, sizeof(int32_t), what, d));
    if (d.rank != 1 || d.ext[0] != B) return fail(ANN_EINVAL, "%s must be rank 1 with one entry per sequence.", what);
    p = static_cast<const int32_t*>(d.data);
    stride = d.str[0];
    return ANN_OK;
}

bool rows4(const Dims& x, size_t elem) {  // unit stride, 4 elements aligned in every row
    if (x.str[3] != 1 || x.ext[3] % 4 != 0 || !aligned(x.data, 4 * elem)) return false;
    return x.str[0] % 4 == 0 && x.str[1] % 4 == 0 && x.str[2] % 4 == 0;
}

int append(ann_stream stream, const ann_view* kn, const ann_view* vn, const ann_view* kc, const ann_view* vc,
           const ann_view* ks, const ann_view* vs, const ann_view* pos_v, const ann_view* counts_v, uint32_t block,
           int layout) {
    char const* what = "kvCacheAppendQ8";
    Dims x[2], q[2], s[2];
    ANN_TRY(to_dims_flat(kn, sizeof(float), what, x[0]));
    ANN_TRY(to_dims_flat(vn, sizeof(float), what, x[1]));
    const ann_view* const qv[2] = {kc, vc};
    const ann_view* const sv[2] = {ks, vs};
    ANN_TRY(cache_tensors(what, qv, sv, block, layout, q, s));
    int const tok = layout == ANN_LAYOUT_BTHD ? 1 : 2, head = 3 - tok;
    if (x[0].rank != 4 || !same_extents(x[0], x[1]))
        return fail(ANN_EINVAL, "kvCacheAppendQ8 expects rank-4 BTHD rows of K and V of the same extents.");
    if (x[0].ext[0] != q[0].ext[0] || x[0].ext[2] != q[0].ext[head] || x[0].ext[3] != q[0].ext[3])
        return fail(ANN_EINVAL, "kvCacheAppendQ8: rows %s do not match the cache %s.", extents_str(x[0]).c_str(),
                    extents_str(q[0]).c_str());
    for (int k = 0; k < 2; ++k)
        if (!writable(q[k]) || !writable(s[k])) return fail(ANN_EINVAL, "kvCacheAppendQ8: a cache axis has a zero pitch.");
    AppendArgs a{};
    int64_t const B = x[0].ext[0];
    ANN_TRY(per_sequence(pos_v, "kvCacheAppendQ8 positions", B, a.pos, a.pos_s));
    if (counts_v != nullptr) ANN_TRY(per_sequence(counts_v, "kvCacheAppendQ8 counts", B, a.counts, a.counts_s));
    a.Tn = x[0].ext[1];
    int64_t const H = x[0].ext[2];
    a.D = x[0].ext[3];
    a.cap = q[0].ext[tok];
    a.block = block;
    if (x[0].numel() == 0) return ANN_OK;
    int64_t const per_block = std::min<int64_t>(block, a.cap) * a.D;
    if (per_block > INT32_MAX - kThreads) return fail(ANN_ENOTSUP, "kvCacheAppendQ8: a block of one head exceeds 2^31 values.");
    a.vec = 1;
    for (int k = 0; k < 2; ++k) {
        a.c[k] = tensor_of(q[k], s[k], layout);
        a.x[k] = static_cast<const float*>(x[k].data);
        a.x_b[k] = x[k].str[0];
        a.x_t[k] = x[k].str[1];
        a.x_h[k] = x[k].str[2];
        a.x_d[k] = x[k].str[3];
        if (!rows4(x[k], sizeof(float)) || !rows4(q[k], 1)) a.vec = 0;
    }
    a.row = FastDiv::make(static_cast<uint32_t>(a.vec ? a.D / 4 : a.D));
    // Threads for eight items each of a block of tokens (8 x 1170 tokens in blocks of 16,
    // 7 heads of 128: 22 us against 42 with 256).
    int64_t const in_block = std::min<int64_t>(block, a.cap) * a.row.d;
    int const threads = in_block <= 512 ? 64 : in_block <= 1024 ? 128 : 256;
    a.rows = static_cast<int>(threads / a.row.d);
    // Rows start anywhere in a block: at most this many blocks hold some of them.
    // (A cache of no tokens has none, and one thread block that reports the rows.)
    int64_t const touched = std::clamp(ceil_div(a.cap, block), int64_t{1}, ceil_div(a.Tn - 1, block) + 1), grid = B * H * 2 * touched;
    if (a.cap > INT32_MAX) return fail(ANN_ENOTSUP, "kvCacheAppendQ8: more than 2^31 tokens.");
    a.touched = FastDiv::make(static_cast<uint32_t>(touched));
    a.heads = FastDiv::make(static_cast<uint32_t>(H));
    a.blocks = FastDiv::make(block);
    if (grid > INT32_MAX) return fail(ANN_ENOTSUP, "kvCacheAppendQ8: grid too large.");
    auto const pick = [&](auto n) {
        constexpr int TH = decltype(n)::value;
        return TH % a.row.d == 0 ? append_kernel<true, TH> : append_kernel<false, TH>;
    };
    auto const kernel = threads == 64    ? pick(std::integral_constant<int, 64>{})
                        : threads == 128 ? pick(std::integral_constant<int, 128>{})
                                         : pick(std::integral_constant<int, 256>{});
    launch_overlapping(kernel, dim3(static_cast<unsigned>(grid)), threads, 0, as_stream(stream), a);
    return check_launch(what);
}

int read_back(ann_stream stream, const ann_view* kc, const ann_view* vc, const ann_view* ks, const ann_view* vs,
              const ann_view* ko, const ann_view* vo, const ann_view* len_v, uint32_t block, int layout) {
    char const* what = "kvCacheReadQ8";
    Dims q[2], s[2], o[2];
    const ann_view* const qv[2] = {kc, vc};
    const ann_view* const sv[2] = {ks, vs};
    ANN_TRY(cache_tensors(what, qv, sv, block, layout, q, s));
    ANN_TRY(to_dims_flat(ko, sizeof(float), what, o[0]));
    ANN_TRY(to_dims_flat(vo, sizeof(float), what, o[1]));
    int const tok = layout == ANN_LAYOUT_BTHD ? 1 : 2, head = 3 - tok;
    for (int k = 0; k < 2; ++k) {
        if (o[k].rank != 4 || o[k].ext[0] != q[k].ext[0] || o[k].ext[head] != q[k].ext[head] ||
            o[k].ext[3] != q[k].ext[3] || o[k].ext[tok] > q[k].ext[tok])
            return fail(ANN_EINVAL, "kvCacheReadQ8: output %s does not match the cache %s.", extents_str(o[k]).c_str(),
                        extents_str(q[k]).c_str());
        if (!writable(o[k])) return fail(ANN_EINVAL, "kvCacheReadQ8: an output axis has a zero pitch.");
    }
    if (!same_extents(o[0], o[1])) return fail(ANN_EINVAL, "kvCacheReadQ8: K and V output extents differ.");
    ReadArgs a{};
    if (len_v != nullptr) ANN_TRY(per_sequence(len_v, "kvCacheReadQ8 lengths", q[0].ext[0], a.lengths, a.len_s));
    int64_t const H = q[0].ext[head];
    a.D = q[0].ext[3];
    a.Tout = o[0].ext[tok];
    if (o[0].numel() == 0) return ANN_OK;
    if (a.Tout > INT32_MAX / a.D - 8 * kThreads) return fail(ANN_ENOTSUP, "kvCacheReadQ8: a head of more than 2^31 values.");
    a.vec = 1;
    for (int k = 0; k < 2; ++k) {
        a.c[k] = tensor_of(q[k], s[k], layout);
        a.out[k] = static_cast<float*>(o[k].data);
        a.o_b[k] = o[k].str[0];
        a.o_h[k] = o[k].str[head];
        a.o_t[k] = o[k].str[tok];
        a.o_d[k] = o[k].str[3];
        if (!rows4(o[k], sizeof(float)) || !rows4(q[k], 1)) a.vec = 0;
    }
    a.row = FastDiv::make(static_cast<uint32_t>(a.vec ? a.D / 4 : a.D));
    a.block = FastDiv::make(block);
    bool const step = kThreads % a.row.d == 0;
    a.rows = kThreads / a.row.d;
    // Eight items a thread where that leaves four blocks an SM and more (4 x 3048
    // tokens, 8 heads of 128: 22.8 us against 27.5; sixteen: 24.5), else four.
    int64_t const heads = q[0].ext[0] * H * 2, items = a.Tout * a.row.d;
    bool const many = heads * ceil_div(items, 8 * kThreads) >= int64_t{4} * sm_count();
    int64_t const chunks = ceil_div(items, (many ? 8 : 4) * kThreads), grid = heads * chunks;
    a.chunks = FastDiv::make(static_cast<uint32_t>(chunks));
    a.heads = FastDiv::make(static_cast<uint32_t>(H));
    if (grid > INT32_MAX) return fail(ANN_ENOTSUP, "kvCacheReadQ8: grid too large.");
    auto const pick = [&](auto each) {
        constexpr int E = decltype(each)::value;
        return a.vec ? (step ? read_kernel<true, true, E> : read_kernel<true, false, E>)
                     : (step ? read_kernel<false, true, E> : read_kernel<false, false, E>);
    };
    auto const kernel = many ? pick(std::integral_constant<int, 8>{}) : pick(std::integral_constant<int, 4>{});
    launch_overlapping(kernel, dim3(static_cast<unsigned>(grid)), kThreads, 0, as_stream(stream), a);
    return check_launch(what);
}

}  // namespace

int take_kv_q8_error(cudaStream_t s, uint32_t* bits) {
    unsigned int value = 0, zero = 0;
    if (cudaMemcpyFromSymbolAsync(&value, g_kv_q8_error, sizeof value, 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
        cudaMemcpyToSymbolAsync(g_kv_q8_error, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, s) != cudaSuccess ||
        cudaStreamSynchronize(s) != cudaSuccess)
        return fail(ANN_ECUDA, "device error word: %s", cudaGetErrorString(cudaGetLastError()));
    *bits |= value;
    return ANN_OK;
}

}  // namespace ann

extern "C" {

int ann_kv_cache_append_q8_f32(ann_stream s, const ann_view* k_new, const ann_view* v_new, const ann_view* k_cache,
                               const ann_view* v_cache, const ann_view* k_scale, const ann_view* v_scale,
                               const ann_view* positions, const ann_view* counts, uint32_t tokens_per_scale,
                               int32_t kv_layout) {
    ANN_API_BEGIN
    return ann::append(s, k_new, v_new, k_cache, v_cache, k_scale, v_scale, positions, counts, tokens_per_scale,
                       kv_layout);
    ANN_API_END
}

int ann_kv_cache_read_q8_f32(ann_stream s, const ann_view* k_cache, const ann_view* v_cache, const ann_view* k_scale,
                             const ann_view* v_scale, const ann_view* k_out, const ann_view* v_out,
                             const ann_view* lengths, uint32_t tokens_per_scale, int32_t kv_layout) {
    ANN_API_BEGIN
    return ann::read_back(s, k_cache, v_cache, k_scale, v_scale, k_out, v_out, lengths, tokens_per_scale, kv_layout);
    ANN_API_END
}

}  // extern "C"
