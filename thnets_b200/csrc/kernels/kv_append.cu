// New tokens' keys and values into a paged cache, the rotation by position on the way, and the same rotation of the queries.
// Pair i of a head (values i and i + dim/2, or 2i and 2i + 1) is turned by the angle pos * freq[i]:
//     a' = (a cos - b sin) * magnitude,  b' = (a sin + b cos) * magnitude.
// pos * freq in fp32 is off by 0.06 rad at a million positions, so the angle is reduced to a fraction of a turn in fp64, once a pair and
// token for all its heads, and cos and sin are taken of that in fp32.  HBM-bound on prompts (each value read and written once),
// latency-bound on a decoder's single tokens.
// us a launch in a chain (share of the measured copy rate), 8192 tokens of 32 + 8 + 8 heads: of 128 in bf16, halves 36.6 (84 %); half of each
// turned in neighbouring pairs, fp16 37.5 (82 %); of 64 23.3 (66 %); 4096 tokens in fp32 34.7 (89 %).  With a block to a token, which
// waits for the angles together: 56 / 47 / 34 / 36.  One unit serves all of a token's values, the unturned ones and v too: with halves that are
// no whole vectors, all travel in 8, 4 or 2 bytes (4096 tokens of 36 heads of 80 in bf16, 40 / 20 / 10 values turned: 22.5 / 41.8 / 57.6, bytes
// alone 7.2).
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

// what a lane moves at a time: 16 bytes where halves and parts of a head allow, else 8, 4 or one value; held as words, so that it is one load
template <int BYTES> struct WordOf;
template <> struct WordOf<16> { using type = uint4; };
template <> struct WordOf<8> { using type = uint2; };
template <> struct WordOf<4> { using type = uint32_t; };
template <> struct WordOf<2> { using type = uint16_t; };
template <typename T, int U> struct Unit {
    typename WordOf<sizeof(T) * U>::type w;
    __device__ __forceinline__ void unpack(float *f) const
    {
        if constexpr (sizeof(T) * U == 16) Vec16<T>::unpack(w, f);
        else
#pragma unroll
            for (int i = 0; i < U; i++) f[i] = dt<T>::ld(reinterpret_cast<const T *>(&w) + i);
    }
    __device__ __forceinline__ void pack(const float *f)
    {
        if constexpr (sizeof(T) * U == 16) w = Vec16<T>::pack(f);
        else
#pragma unroll
            for (int i = 0; i < U; i++) dt<T>::st(reinterpret_cast<T *>(&w) + i, f[i]);
    }
};

// A warp has every parts-th group of `slots` heads of a token, on its own: where there are many tokens one warp has all heads, so that angles
// are taken once, where there are few several share them.  A lane has the same item of each of its heads: a pair of units of both halves, a
// unit of neighbouring pairs, or units that are not turned; the angles it turns by stay in its registers.  HEADS of them are under way, the
// first before the position and the page are known.
// How many heads, and blocks an SM.  Halves in whole units: few warps with many loads each (8192 tokens of 32 + 8 + 8 heads of 128 in bf16, 6 and
// two blocks against 4 and two: 36.6 us for 39.8).  Pairs, or smaller units, take more instructions a byte: fewer loads, more warps (half of each
// head in pairs, fp16, 3 and four against 4 and three: 37.5 for 40.3; 4096 tokens of 36 heads of 80 in units of 8 bytes, 2 and four against 4 and
// three: 22.0 for 35.7).  Halves of an odd number of values, taken one by one, 2 and four against 4 and three: 4096 tokens of 36 heads of 80 with 10 values
// turned 57.6 for 62.6 in bf16, 57.7 for 67.3 in fp32, 512 of them 10.6 for 12.2; 8192 of 48 heads of 128 with 18 turned 170 for 163.
template <typename T, int U, bool INTER> struct AppendShape {
    static constexpr bool MANY = !INTER && sizeof(T) * U == 16;
    static constexpr int HEADS = INTER ? 3 : MANY ? 6 : 2, BLOCKS = MANY ? 2 : 4;
};
template <typename T, int U, bool INTER>
__global__ void __launch_bounds__(256, (AppendShape<T, U, INTER>::BLOCKS)) kv_append_kernel(AppendParams p, int items, int per, int slots, int parts)
{
    constexpr int HEADS = AppendShape<T, U, INTER>::HEADS, PAIRS = INTER ? U / 2 : U;  // pairs an item
    __shared__ float2 turns_of[8][128];
    pdl_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long mine = (long)blockIdx.x * 8 + warp;
    const int token = (int)(mine / parts), part = (int)(mine % parts);
    if (token >= p.tokens) return;
    const int pos = p.pos[token], seq = p.k && p.seq ? p.seq[token] : token;
    const int rot = p.rope.dim, half = rot / 2, dim = p.c.dim, turned = INTER ? rot / U : half / U;
    const int nq = p.q ? p.q_heads : 0, nk = p.k ? p.c.heads : 0, heads = nq + 2 * nk;
    const T *const q = (const T *)p.q + (long)token * p.q_ld, *const k = (const T *)p.k + (long)token * p.k_ld, *const v = (const T *)p.v + (long)token * p.v_ld;
    T *const q_out = (T *)p.q_out + (long)token * p.q_out_ld, *ck = nullptr, *cv = nullptr;
    float2 *const turn = turns_of[warp];
    bool known = false;

    for (int item0 = 0; item0 < items; item0 += per) {
        const int item = item0 + lane % per, sub = lane / per;
        const bool turns = item < turned, working = item < items && sub < slots;
        // the item's first values, and those `apart` behind them where it has two units
        const int at = turns ? item * U : rot + (item - turned) * U;
        const int apart = turns && !INTER ? half : 0;
        float2 w[PAIRS];
        for (int h0 = part * slots + sub; h0 - sub < heads; h0 += HEADS * slots * parts) {
            Unit<T, U> a[HEADS], b[HEADS];
#pragma unroll
            for (int i = 0; i < HEADS; i++) {
                const int h = h0 + i * slots * parts;
                if (!working || h >= heads) break;
                const T *from = (h < nq ? q + h * dim : h < nq + nk ? k + (h - nq) * dim : v + (h - nq - nk) * dim) + at;
                a[i] = *reinterpret_cast<const Unit<T, U> *>(from);
                if (apart) b[i] = *reinterpret_cast<const Unit<T, U> *>(from + apart);
            }
            if (!known) {
                if (pos < 0) return;  // a place in a padded batch
                // the token's place: anything beyond the table or the pool is not written
                if (p.k) {
                    const int slot = pos / p.c.page_len;
                    int page = -1;
                    if ((unsigned)seq < (unsigned)p.c.sequences && slot < p.c.table_ld) page = p.c.table[(long)seq * p.c.table_ld + slot];
                    if ((unsigned)page < (unsigned)p.c.pages) {
                        const long place = page * p.c.page_stride + (pos - slot * p.c.page_len) * p.c.token_stride;
                        ck = (T *)p.c.k + place;
                        cv = (T *)p.c.v + place;
                    } else if (lane == 0)
                        *p.c.status = THB_ERR_ARG;
                }
                for (int i = lane; i < half; i += 32) {
                    double t = (double)pos * p.rope.freq[i] * 0.15915494309189533577;  // in turns
                    t -= rint(t);
                    float sn, cs;
                    sincospif((float)(2 * t), &sn, &cs);
                    turn[i] = make_float2(cs * p.rope.magnitude, sn * p.rope.magnitude);
                }
                __syncwarp();
                known = true;
            }
            if (h0 == part * slots + sub)
#pragma unroll
                for (int j = 0; j < PAIRS; j++) w[j] = turns ? turn[item * PAIRS + j] : make_float2(1.f, 0.f);
#pragma unroll
            for (int i = 0; i < HEADS; i++) {
                const int h = h0 + i * slots * parts;
                if (!working || h >= heads) break;
                T *to = h < nq ? q_out + h * dim : ck == nullptr ? nullptr : h < nq + nk ? ck + (h - nq) * p.c.head_stride : cv + (h - nq - nk) * p.c.head_stride;
                if (to == nullptr) break;  // (the queries come first)
                if (turns && h < nq + nk) {
                    float x[U], y[U];
                    a[i].unpack(x);
                    if constexpr (!INTER) {
                        b[i].unpack(y);
#pragma unroll
                        for (int j = 0; j < U; j++) {
                            const float r = x[j] * w[j].x - y[j] * w[j].y;
                            y[j] = x[j] * w[j].y + y[j] * w[j].x;
                            x[j] = r;
                        }
                        b[i].pack(y);
                    } else {
#pragma unroll
                        for (int j = 0; j < U; j += 2) {
                            const float r = x[j] * w[j / 2].x - x[j + 1] * w[j / 2].y;
                            x[j + 1] = x[j] * w[j / 2].y + x[j + 1] * w[j / 2].x;
                            x[j] = r;
                        }
                    }
                    a[i].pack(x);
                }
                *reinterpret_cast<Unit<T, U> *>(to + at) = a[i];
                if (apart) *reinterpret_cast<Unit<T, U> *>(to + at + apart) = b[i];
            }
        }
    }
}

template <typename T, int U> int launch_units(const AppendParams &p, cudaStream_t st)
{
    const int rot = p.rope.dim, half = rot / 2, dim = p.c.dim, heads = (p.q ? p.q_heads : 0) + (p.k ? 2 * p.c.heads : 0);
    const bool inter = p.rope.interleaved;
    // a head's items, taken at most 32 at a time
    const int items = (inter ? rot / U : half / U) + (dim - rot) / U, turns = (items + 31) / 32, per = (items + turns - 1) / turns, slots = 32 / per;
    // a warp a token where there are enough of them for 16 warps an SM; else as many as that takes, with a few heads each
    long parts = 1;
    const int most = (heads + slots - 1) / slots;
    while (parts * 2 <= most && p.tokens * parts < 16L * thb_sm_count()) parts *= 2;
    const unsigned grid = (unsigned)((p.tokens * parts + 7) / 8);
    if (!inter) thb_launch(kv_append_kernel<T, U, false>, grid, 256, st, p, items, per, slots, (int)parts);
    else if constexpr (U > 1) thb_launch(kv_append_kernel<T, U, true>, grid, 256, st, p, items, per, slots, (int)parts);  // (pairs are whole in units of two)
    return THB_LAUNCH_CHECK("kv_append_kernel");
}

template <typename T> int launch_append(const AppendParams &p, cudaStream_t st)
{
    constexpr int VN = Vec16<T>::N;
    const int unit = p.rope.interleaved ? p.rope.dim : p.rope.dim / 2;  // what whole units have to make up (0: nothing is turned)
    if (unit % VN == 0) return launch_units<T, VN>(p, st);
    if constexpr (VN == 8)
        if (unit % 4 == 0) return launch_units<T, 4>(p, st);
    if (unit % 2 == 0) return launch_units<T, 2>(p, st);
    return launch_units<T, 1>(p, st);
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
    if (q && q == q_out && d->tokens > 1 && d->q_ld != d->q_out_ld) return thb_refuse(THB_ERR_ARG, "thb_kv_append_fwd: q_out in the place of q with another ld");
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
