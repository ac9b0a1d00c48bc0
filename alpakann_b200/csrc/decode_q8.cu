// decode_q8.cu -- attention of the last tokens over a KV cache held in 8 bits.
//
// Query i of Tq (the last tokens of a sequence of `length` keys) and head hq:
//   s_j = scale * ks[j / block] * (q . n_j),  j < length - Tq + 1 + i  (causal) or j < length
//   out = sum_j e^(s_j - max s) vs[j / block] m_j / sum_j e^(s_j - max s)
// with n_j, m_j the cache's whole numbers (kv_q8.cu). A query that sees no key
// gets a row of zeros.
#include <algorithm>

#include "common.cuh"
#include "reduce.cuh"

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
    int block_shift, causal;
    float scale;
};

constexpr int kThreads = 128;

// One block per query row: 128 keys at a time, a thread per key for the scores
// and a thread per head element for the sum.
template <int D>
__global__ void __launch_bounds__(kThreads) decode_q8_kernel(DecodeQ8Args a) {
    __shared__ float qs[D];
    __shared__ float ps[kThreads];
    __shared__ float red[kThreads / 32];
    int const tid = threadIdx.x;
    int64_t const hq = blockIdx.x % a.Hq, tq = (blockIdx.x / a.Hq) % a.Tq, b = blockIdx.x / (a.Hq * a.Tq);
    int64_t const kvh = hq / a.g;
    int64_t len = a.cap;
    if (a.lengths != nullptr) len = min(a.cap, max(int64_t{0}, static_cast<int64_t>(a.lengths[b * a.len_s])));
    if (a.causal) len = len - a.Tq + 1 + tq;
    float const* q = a.q + b * a.q_b + tq * a.q_t + hq * a.q_h;
    for (int d = tid; d < D; d += kThreads) qs[d] = q[d];
    int8_t const* kb = a.k + b * a.k_b + kvh * a.k_h;
    int8_t const* vb = a.v + b * a.v_b + kvh * a.v_h;
    float const* ks = a.ks + b * a.ks_b + kvh * a.ks_h;
    float const* vs = a.vs + b * a.vs_b + kvh * a.vs_h;
    float m = neg_inf(0.0f), l = 0.0f;
    constexpr int E = (D + kThreads - 1) / kThreads;
    float o[E] = {};
    __syncthreads();
    for (int64_t j0 = 0; j0 < len; j0 += kThreads) {
        int64_t const j = j0 + tid;
        float s = neg_inf(0.0f);
        if (j < len) {
            int8_t const* row = kb + j * a.k_t;
            float acc = 0.0f;
            for (int d = 0; d < D; d += 16) {
                int4 const w = *reinterpret_cast<int4 const*>(row + d);
                int const ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc = fmaf(qs[d + e], static_cast<float>(static_cast<int8_t>(ws[e / 4] >> (8 * (e % 4)))), acc);
            }
            s = acc * ks[(j >> a.block_shift) * a.ks_j] * a.scale;
        }
        float const m_new = fmaxf(m, block_max<kThreads / 32>(s, red));
        float const base = m_new == neg_inf(0.0f) ? 0.0f : m_new;
        float const p = j < len ? expf(s - base) : 0.0f, alpha = expf(m - base);
        l = l * alpha + block_sum<kThreads / 32>(p, red);
        m = m_new;
        ps[tid] = j < len ? p * vs[(j >> a.block_shift) * a.vs_j] : 0.0f;
        __syncthreads();
        int const n = static_cast<int>(min(int64_t{kThreads}, len - j0));
#pragma unroll
        for (int e = 0; e < E; ++e) {
            int const d = tid + e * kThreads;
            o[e] *= alpha;
            if (d < D)
                for (int i = 0; i < n; ++i) o[e] = fmaf(ps[i], static_cast<float>(vb[(j0 + i) * a.v_t + d]), o[e]);
        }
        __syncthreads();
    }
    float* out = a.out + b * a.o_b + tq * a.o_t + hq * a.o_h;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        int const d = tid + e * kThreads;
        if (d < D) out[d * a.o_d] = l == 0.0f ? 0.0f : o[e] / l;
    }
}

template <int D>
int launch(ann_stream stream, DecodeQ8Args const& a) {
    int64_t const grid = a.B * a.Tq * a.Hq;
    if (grid > INT32_MAX) return fail(ANN_ENOTSUP, "attentionDecodeQ8: grid too large.");
    decode_q8_kernel<D><<<static_cast<unsigned>(grid), kThreads, 0, as_stream(stream)>>>(a);
    return check_launch("attentionDecodeQ8");
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
    a.B = B;
    a.Tq = q.ext[1];
    a.Hq = Hq;
    a.Hkv = k.ext[head];
    a.cap = k.ext[tok];
    a.g = g;
    a.block_shift = __builtin_ctz(block);
    a.causal = causal != 0;
    a.scale = scale;
    if (D == 64) return launch<64>(stream, a);
    if (D == 128) return launch<128>(stream, a);
    return launch<256>(stream, a);
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
