// New tokens' keys and values into a paged cache, the rotation by position on the way, and the same rotation of the queries.
// Pair i of a head (values i and i + dim/2, or 2i and 2i + 1) is turned by the angle pos * freq[i]:
//     a' = (a cos - b sin) * magnitude,  b' = (a sin + b cos) * magnitude.
// pos * freq in fp32 is off by 0.06 rad at a million positions, so the angle is reduced to a fraction of a turn in fp64, once a pair and
// token for all its heads, and cos and sin are taken of that in fp32.  HBM-bound on prompts (each value read and written once),
// latency-bound on a decoder's single tokens.
#include "tokens.cuh"
#include <math.h>

namespace {

struct AppendParams {
    thb_kv_cache c;
    thb_rope rope;
    const int *pos, *seq;
    const void *k, *v, *q;
    void *q_out;
    int tokens, q_heads, k_ld, v_ld, q_ld, q_out_ld;
};

template <typename T, int U> __device__ __forceinline__ void get(const T *p, float *v)
{
    if constexpr (U == 1) v[0] = dt<T>::ld(p);
    else Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(p), v);
}
template <typename T, int U> __device__ __forceinline__ void put(T *p, const float *v)
{
    if constexpr (U == 1) dt<T>::st(p, v[0]);
    else *reinterpret_cast<uint4 *>(p) = Vec16<T>::pack(v);
}

// A block has a token.  U: values an access, 16 bytes of them, or one where a vector would hold values of both halves of a pair's
// or of the rotated and the other part of a head.
template <typename T, int U>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendParams p)
{
    __shared__ float2 turn[128];
    pdl_enter();
    const int token = blockIdx.x, pos = p.pos[token];
    if (pos < 0) return;  // a place in a padded batch
    const int rot = p.rope.dim, half = rot / 2, dim = p.c.dim;
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        double t = (double)pos * p.rope.freq[i] * 0.15915494309189533577;  // in turns
        t -= rint(t);
        float sn, cs;
        sincospif((float)(2 * t), &sn, &cs);
        turn[i] = make_float2(cs * p.rope.magnitude, sn * p.rope.magnitude);
    }
    // the token's place: anything beyond the table or the pool is not written
    T *ck = nullptr, *cv = nullptr;
    if (p.k) {
        const int seq = p.seq ? p.seq[token] : token, slot = pos / p.c.page_len;
        int page = -1;
        if ((unsigned)seq < (unsigned)p.c.sequences && slot < p.c.table_ld) page = p.c.table[(long)seq * p.c.table_ld + slot];
        if ((unsigned)page < (unsigned)p.c.pages) {
            const long at = page * p.c.page_stride + (pos - slot * p.c.page_len) * p.c.token_stride;
            ck = (T *)p.c.k + at;
            cv = (T *)p.c.v + at;
        } else if (threadIdx.x == 0)
            *p.c.status = THB_ERR_ARG;
    }
    __syncthreads();

    // a head's items: pairs of vectors (halves) or vectors of pairs (neighbours) that are turned, then vectors that are copied
    const int turned = p.rope.interleaved ? (U == 1 ? half : rot / U) : half / U, items = turned + (dim - rot) / U, copied = dim / U;
    auto rotate = [&](const T *src, T *dst, int item) {
        float a[U], b[U];
        if (item >= turned) {
            const int o = rot + (item - turned) * U;
            get<T, U>(src + o, a);
            put<T, U>(dst + o, a);
        } else if (!p.rope.interleaved) {
            const int o = item * U;
            get<T, U>(src + o, a);
            get<T, U>(src + o + half, b);
#pragma unroll
            for (int j = 0; j < U; j++) {
                const float2 w = turn[o + j];
                const float x = a[j], y = b[j];
                a[j] = x * w.x - y * w.y;
                b[j] = x * w.y + y * w.x;
            }
            put<T, U>(dst + o, a);
            put<T, U>(dst + o + half, b);
        } else if constexpr (U == 1) {
            const float2 w = turn[item];
            const float x = dt<T>::ld(src + 2 * item), y = dt<T>::ld(src + 2 * item + 1);
            dt<T>::st(dst + 2 * item, x * w.x - y * w.y);
            dt<T>::st(dst + 2 * item + 1, x * w.y + y * w.x);
        } else {
            const int o = item * U;
            get<T, U>(src + o, a);
#pragma unroll
            for (int j = 0; j < U; j += 2) {
                const float2 w = turn[(o + j) / 2];
                const float x = a[j], y = a[j + 1];
                a[j] = x * w.x - y * w.y;
                a[j + 1] = x * w.y + y * w.x;
            }
            put<T, U>(dst + o, a);
        }
    };
    const int nq = p.q ? p.q_heads * items : 0, nk = ck ? p.c.heads * items : 0, nv = ck ? p.c.heads * copied : 0;
    for (int i = threadIdx.x; i < nq + nk + nv; i += blockDim.x) {
        if (i < nq) {
            const int h = i / items;
            rotate((const T *)p.q + (long)token * p.q_ld + h * dim, (T *)p.q_out + (long)token * p.q_out_ld + h * dim, i - h * items);
        } else if (i < nq + nk) {
            const int h = (i - nq) / items;
            rotate((const T *)p.k + (long)token * p.k_ld + h * dim, ck + h * p.c.head_stride, i - nq - h * items);
        } else {
            const int h = (i - nq - nk) / copied, o = (i - nq - nk - h * copied) * U;
            float a[U];
            get<T, U>((const T *)p.v + (long)token * p.v_ld + h * dim + o, a);
            put<T, U>(cv + h * p.c.head_stride + o, a);
        }
    }
}

template <typename T> int launch_append(const AppendParams &p, cudaStream_t st)
{
    constexpr int VN = Vec16<T>::N;
    const bool vectors = (p.rope.interleaved ? p.rope.dim : p.rope.dim / 2) % VN == 0;
    if (vectors) thb_launch(kv_append_kernel<T, VN>, (unsigned)p.tokens, 256, st, p);
    else thb_launch(kv_append_kernel<T, 1>, (unsigned)p.tokens, 256, st, p);
    return THB_LAUNCH_CHECK("kv_append_kernel");
}

}  // namespace

// What a cache's descriptor has to be, whoever uses it; NULL: nothing is wrong.
const char *thb_kv_cache_fault(const thb_kv_cache *c)
{
    const int al = thb_channel_align(c->dtype);
    if (c->heads < 1 || c->dim < al || c->dim % al || c->dim > 256) return "KV cache: heads below 1, or dim no multiple of the alignment or above 256";
    if (c->pages < 1 || c->page_len < 1 || c->table_ld < 1 || c->sequences < 1) return "KV cache: pages, page_len, table_ld or sequences below 1";
    if (!c->k || !c->v || !c->table || !c->status) return "KV cache: k, v, table and status must be set";
    if (thb_misaligned(c->k) || thb_misaligned(c->v)) return "KV cache: k or v is not 16-byte aligned";
    if (c->page_stride < 0 || c->token_stride < 0 || c->head_stride < 0 || c->page_stride % al || c->token_stride % al || c->head_stride % al)
        return "KV cache: a stride is negative or no multiple of the alignment";
    // tokens and heads of a page have places of their own, whichever of the two is the inner one (a single one has no stride)
    const long heads = c->heads - 1, tokens = c->page_len - 1, most = 1L << 40;
    if (c->page_stride > most || c->token_stride > most / c->page_len || c->head_stride > most / c->heads) return "KV cache: a stride is too large";
    const bool by_token = (!heads || c->head_stride >= c->dim) && (!tokens || c->token_stride >= heads * c->head_stride + c->dim);
    const bool by_head = (!tokens || c->token_stride >= c->dim) && (!heads || c->head_stride >= tokens * c->token_stride + c->dim);
    if (!by_token && !by_head) return "KV cache: tokens or heads of a page overlap";
    if (c->pages > 1 && c->page_stride < tokens * c->token_stride + heads * c->head_stride + c->dim) return "KV cache: pages overlap";
    return nullptr;
}

extern "C" int thb_kv_append_fwd(const thb_kv_append_desc *d, const void *k, const void *v, const void *q, void *q_out, thb_stream s)
{
    if (!d) return THB_ERR_ARG;
    const int dtype = d->cache.dtype;
    if (dtype != THB_F32 && dtype != THB_F16 && dtype != THB_BF16)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_kv_append_fwd: dtype is not THB_F32, THB_F16 or THB_BF16");
    if (d->tokens < 0) return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: tokens < 0");
    if (d->tokens == 0) return THB_OK;
    const int al = thb_channel_align(dtype), dim = d->cache.dim;
    if (!k != !v || !q != !q_out || (!k && !q) || !d->pos) return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: k with v, q with q_out, one pair at least, and pos must be set");
    if (k) {
        const char *why = thb_kv_cache_fault(&d->cache);
        if (why) return thb_refuse(THB_ERR_ARG, why);
        if (!d->seq && d->tokens > d->cache.sequences) return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: more tokens than sequences, and no seq");
    } else if (dim < al || dim % al || dim > 256)
        return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: dim is no multiple of the alignment or above 256");
    if (d->rope.dim < 0 || d->rope.dim % 2 || d->rope.dim > dim || (d->rope.dim && !d->rope.freq))
        return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: rope.dim is negative, odd or above dim, or freq is missing");
    const long kw = (long)d->cache.heads * dim, qw = (long)d->q_heads * dim;
    if (q && (d->q_heads < 1 || d->q_ld < qw || d->q_out_ld < qw || d->q_ld % al || d->q_out_ld % al || thb_misaligned(q) || thb_misaligned(q_out)))
        return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: q_heads < 1, q or q_out not 16-byte aligned, or q_ld or q_out_ld below the row or no multiple of the alignment");
    if (k && (d->k_ld < kw || d->v_ld < kw || d->k_ld % al || d->v_ld % al || thb_misaligned(k) || thb_misaligned(v)))
        return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: k or v not 16-byte aligned, or k_ld or v_ld below the row or no multiple of the alignment");
    // (a row's items are counted in 32 bits)
    if (qw + 2 * kw > (1L << 30)) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_kv_append_fwd: heads of more than 2^30 values a token");
    const AppendParams p = {d->cache, d->rope, d->pos, d->seq, k, v, q, q_out, d->tokens, d->q_heads, d->k_ld, d->v_ld, d->q_ld, d->q_out_ld};
    switch (dtype) {
    case THB_F32: return launch_append<float>(p, (cudaStream_t)s);
    case THB_F16: return launch_append<__half>(p, (cudaStream_t)s);
    default: return launch_append<__nv_bfloat16>(p, (cudaStream_t)s);
    }
}

extern "C" int thb_rope_freq_host(int dim, double base, int scaling, double factor, double trained_len, double slow_turns, double fast_turns,
                                  double *freq_host, float *magnitude)
{
    if (dim < 2 || dim % 2 || !(base > 0) || !freq_host || !magnitude) return THB_ERR_ARG;
    if (scaling < THB_ROPE_PLAIN || scaling > THB_ROPE_BY_PARTS) return THB_ERR_UNSUPPORTED;
    if (scaling != THB_ROPE_PLAIN && !(factor >= 1 && factor < 1e9)) return THB_ERR_ARG;
    if (scaling == THB_ROPE_BASE && dim == 2) return THB_ERR_UNSUPPORTED;  // its one pair does not depend on the base
    if (scaling == THB_ROPE_BY_PARTS && !(trained_len > 0 && slow_turns >= 0 && fast_turns > slow_turns)) return THB_ERR_ARG;
    *magnitude = 1.f;
    if (scaling == THB_ROPE_BASE) base *= pow(factor, (double)dim / (dim - 2));
    for (int i = 0; i < dim / 2; i++) {
        double f = pow(base, -2.0 * i / dim);
        if (scaling == THB_ROPE_LINEAR) f /= factor;
        if (scaling == THB_ROPE_BY_PARTS) {
            const double turns = trained_len * f * 0.15915494309189533577;
            double keep = (turns - slow_turns) / (fast_turns - slow_turns);
            keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * keep + f / factor * (1 - keep);
        }
        freq_host[i] = f;
    }
    if (scaling == THB_ROPE_BY_PARTS) *magnitude = (float)(0.1 * log(factor) + 1.0);
    return THB_OK;
}
