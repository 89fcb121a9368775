// Attention of one new token a sequence over a paged cache: y_h = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q_h.k_j - max), over the
// positions j of [max(0, len - window), len).
// HBM-bound on the cache: 4 * heads / kv_heads operations for every 2 values read.  One pass with a running maximum and sum; both
// products run on the tensor cores (mma.sync m16n8k16: 16 tokens or 16 values of a head by the 8 query heads that share a key
// head; tcgen05's 128-row tiles would be mostly empty), with operands as they are loaded: no shared memory between HBM and the
// registers, bytes in flight come from many warps.
//   S^T[16 tokens][8 heads] = K Q^T:  lane (g = lane / 4, t = lane % 4) holds tokens g and g + 8, 16 bytes at value 4t or 8t of each
//                                     64-byte piece; the order of the values in a product is free, Q takes the same.
//   O^T[16 values][8 heads] = V^T P^T: lane (g, t) holds tokens 2t, 2t + 1, 2t + 8, 2t + 9, 16 bytes at g of each 128-byte piece; bytes of
//                                     two tokens are paired by byte permutes, P by a transposing move.
// 16-bit types: p is two parts (its nearest value and what is left), so that its rounding does not show; fp32: k, q, v and p are three bf16
// parts each (8 + 8 + 8 bits), the six products above 2^-24 are added.
// The length is split among CTAs by `chunk` tokens and joined by a second launch.
#include "tokens.cuh"
#include <math.h>

namespace {

struct AttnParams {
    thb_kv_cache c;
    const int *len, *seq;
    const void *q;
    void *y;
    float *lse, *part;
    int rows, q_heads, q_ld, y_ld, max_len, window, share, head_tiles, chunk, chunks;
    float scale;
};

constexpr int WARPS = 4;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// fp16 holds p only down to 2^-24: there it is p * 2^12, which the division by the sum takes back
template <typename T> constexpr float SHIFT = 0.f;
template <> constexpr float SHIFT<__half> = 12.f;

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint4 load_once(const void *p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// three parts of an fp32 value, each in the top 16 bits of a word
__device__ __forceinline__ void parts_of(uint32_t x, uint32_t (&p)[3])
{
    p[0] = x;
#pragma unroll
    for (int i = 1; i < 3; i++) {
        const float v = __uint_as_float(p[i - 1]), top = __uint_as_float(p[i - 1] & 0xffff0000u);
        p[i] = __float_as_uint(v == top ? 0.f : v - top);  // (an infinity's rest is zero, not NaN)
    }
}
__device__ __forceinline__ uint32_t tops(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

template <typename T> __device__ __forceinline__ uint32_t pair16(float a, float b);
template <> __device__ __forceinline__ uint32_t pair16<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pair16<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T> __device__ __forceinline__ float2 wide16(uint32_t u);
template <> __device__ __forceinline__ float2 wide16<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
template <> __device__ __forceinline__ float2 wide16<__nv_bfloat16>(uint32_t u)
{
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// the positions of a row: [first, last); last < first: a place in a padded batch
__device__ __forceinline__ void positions(const AttnParams &p, int row, int &first, int &last)
{
    last = p.len[row];
    first = 0;
    if (last < 0) {
        last = -1;
        return;
    }
    const long table = (long)p.c.table_ld * p.c.page_len;
    const int most = table < p.max_len ? (int)table : p.max_len, seq = p.seq ? p.seq[row] : row;
    if (last > most || (unsigned)seq >= (unsigned)p.c.sequences) {
        *p.c.status = THB_ERR_ARG;
        last = (unsigned)seq < (unsigned)p.c.sequences ? most : 0;
    }
    if (p.window && last > p.window) first = last - p.window;
}

template <typename T, int DP>
__global__ void __launch_bounds__(WARPS * 32) paged_attn_kernel(AttnParams p)
{
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int VN = Vec16<T>::N;
    constexpr int KV = DP / (4 * VN);      // 16-byte pieces of a token's key that a lane holds
    constexpr int VV = DP / (8 * VN);      // and of a value
    constexpr int QW = F32 ? 6 : 4;        // words of Q beside a piece
    constexpr int TILES = DP / 16;
    __shared__ uint32_t qs[KV][QW][32];
    __shared__ float os[WARPS][8][DP];
    __shared__ float ms[WARPS][8], ls[WARPS][8];
    pdl_enter();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, dim = p.c.dim;
    const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
    const int kv_head = blockIdx.y / p.head_tiles, head0 = (blockIdx.y % p.head_tiles) * 8, heads = min(8, p.share - head0);
    const int q_head0 = kv_head * p.share + head0;
    int first, last;
    positions(p, row, first, last);
    if (last < first) return;
    const int begin = first + chunk * p.chunk, end = min(last, begin + p.chunk);
    if (begin >= last && (chunk > 0 || p.chunks > 1)) return;

    const int seq = p.seq ? p.seq[row] : row;
    const int *table = p.c.table + (long)((unsigned)seq < (unsigned)p.c.sequences ? seq : 0) * p.c.table_ld;
    auto page_of = [&](int token) { return token < end ? table[token / p.c.page_len] : 0; };
    int page = page_of(begin + warp * 16 + (lane & 15));

    // Q beside the keys' pieces
    for (int j = warp; j < KV; j += WARPS) {
        const int d = (j * 4 + t) * VN;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (g < heads && d < dim) v = *reinterpret_cast<const uint4 *>((const T *)p.q + (long)row * p.q_ld + (long)(q_head0 + g) * dim + d);
        if (F32) {
            uint32_t a[4][3];
            parts_of(v.x, a[0]); parts_of(v.y, a[1]); parts_of(v.z, a[2]); parts_of(v.w, a[3]);
#pragma unroll
            for (int i = 0; i < 3; i++) {
                qs[j][(2 * i) % QW][lane] = tops(a[0][i], a[1][i]);
                qs[j][(2 * i + 1) % QW][lane] = tops(a[2][i], a[3][i]);
            }
        } else {
            qs[j][0][lane] = v.x; qs[j][1][lane] = v.y; qs[j][2][lane] = v.z; qs[j][3][lane] = v.w;
        }
    }
    __syncthreads();

    float o[TILES][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[i][k] = 0.f;
    const float scale = p.scale * LOG2E;
    const long head_at = kv_head * p.c.head_stride;

    for (int tile = begin + warp * 16; tile < end; tile += WARPS * 16) {
        // where this tile's tokens lie; the pages of the next are on their way
        const int token = tile + (lane & 15);
        const bool there = (unsigned)page < (unsigned)p.c.pages, ok = token < end && there;
        if (token < end && !there) *p.c.status = THB_ERR_ARG;
        const long at = ok ? page * p.c.page_stride + (token % p.c.page_len) * p.c.token_stride + head_at : -1;
        page = page_of(token + WARPS * 16);
        uint4 kb[2][KV], vb[4][VV];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const long a = __shfl_sync(0xffffffffu, at, g + 8 * r);
#pragma unroll
            for (int j = 0; j < KV; j++) {
                const int d = (j * 4 + t) * VN;
                kb[r][j] = make_uint4(0, 0, 0, 0);
                if (a >= 0 && d < dim) kb[r][j] = load_once((const T *)p.c.k + a + d);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const long a = __shfl_sync(0xffffffffu, at, 2 * t + (r & 1) + 8 * (r >> 1));
#pragma unroll
            for (int j = 0; j < VV; j++) {
                const int d = (j * 8 + g) * VN;
                vb[r][j] = make_uint4(0, 0, 0, 0);
                if (a >= 0 && d < dim) vb[r][j] = load_once((const T *)p.c.v + a + d);
            }
        }
        const uint32_t seen = __ballot_sync(0xffffffffu, ok);

        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KV; j++) {
            const uint4 a = kb[0][j], b = kb[1][j];
            if constexpr (F32) {
                uint32_t x[4][3], y[4][3];
                parts_of(a.x, x[0]); parts_of(a.y, x[1]); parts_of(a.z, x[2]); parts_of(a.w, x[3]);
                parts_of(b.x, y[0]); parts_of(b.y, y[1]); parts_of(b.z, y[2]); parts_of(b.w, y[3]);
#pragma unroll
                for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                    for (int i = sum; i >= 0; i--)
                        mma<T>(s, tops(x[0][i], x[1][i]), tops(y[0][i], y[1][i]), tops(x[2][i], x[3][i]), tops(y[2][i], y[3][i]),
                               qs[j][(2 * (sum - i)) % QW][lane], qs[j][(2 * (sum - i) + 1) % QW][lane]);
            } else {
                mma<T>(s, a.x, b.x, a.y, b.y, qs[j][0][lane], qs[j][1][lane]);
                mma<T>(s, a.z, b.z, a.w, b.w, qs[j][2][lane], qs[j][3][lane]);
            }
        }
        // the softmax's running maximum and sum of heads 2t and 2t + 1; a lane has tokens g and g + 8 of the sum
        const bool see0 = seen >> g & 1, see1 = seen >> (g + 8) & 1;
        float pr[4], shrink[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float a = see0 ? s[h] * scale : -INFINITY, b = see1 ? s[2 + h] * scale : -INFINITY;
            float top = fmaxf(a, b);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top, m[h]);
            const float ref = top == -INFINITY ? 0.f : top;  // (nothing seen yet: every p is zero)
            shrink[h] = exp2f(m[h] - ref);
            m[h] = top;
            pr[h] = exp2f(a - ref + SHIFT<T>);
            pr[2 + h] = exp2f(b - ref + SHIFT<T>);
            l[h] = l[h] * shrink[h] + (pr[h] + pr[2 + h]);
        }
        if (__any_sync(0xffffffffu, shrink[0] != 1.f || shrink[1] != 1.f))
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                o[i][0] *= shrink[0]; o[i][1] *= shrink[1]; o[i][2] *= shrink[0]; o[i][3] *= shrink[1];
            }
        // p as the B operand: parts of (token, heads 2t, 2t + 1), transposed to (head, tokens 2t, 2t + 1)
        constexpr int PP = F32 ? 3 : 2;
        uint32_t pb[PP][2];
        if constexpr (F32) {
            uint32_t x[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++) parts_of(__float_as_uint(pr[i]), x[i]);
#pragma unroll
            for (int i = 0; i < 3; i++) {
                pb[i][0] = transpose8x8(tops(x[0][i], x[1][i]));
                pb[i][1] = transpose8x8(tops(x[2][i], x[3][i]));
            }
        } else {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint32_t u = pair16<T>(pr[2 * r], pr[2 * r + 1]);
                const float2 w = wide16<T>(u);
                pb[0][r] = transpose8x8(u);
                pb[1][r] = transpose8x8(pair16<T>(pr[2 * r] - w.x, pr[2 * r + 1] - w.y));
            }
        }
#pragma unroll
        for (int j = 0; j < VV; j++) {
            uint32_t w[4][4];
#pragma unroll
            for (int r = 0; r < 4; r++) { w[r][0] = vb[r][j].x; w[r][1] = vb[r][j].y; w[r][2] = vb[r][j].z; w[r][3] = vb[r][j].w; }
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 2; i++) {  // values 2i and 2i + 1 of the piece
                    uint32_t x[4][2][3];
#pragma unroll
                    for (int r = 0; r < 4; r++) { parts_of(w[r][2 * i], x[r][0]); parts_of(w[r][2 * i + 1], x[r][1]); }
#pragma unroll
                    for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                        for (int a = sum; a >= 0; a--)
                            mma<T>(o[j * 2 + i], tops(x[0][0][a], x[1][0][a]), tops(x[0][1][a], x[1][1][a]), tops(x[2][0][a], x[3][0][a]),
                                   tops(x[2][1][a], x[3][1][a]), pb[sum - a][0], pb[sum - a][1]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5410), a1 = __byte_perm(w[0][i], w[1][i], 0x7632);
                    const uint32_t a2 = __byte_perm(w[2][i], w[3][i], 0x5410), a3 = __byte_perm(w[2][i], w[3][i], 0x7632);
                    mma<T>(o[(j * 4 + i) % TILES], a0, a1, a2, a3, pb[1][0], pb[1][1]);
                    mma<T>(o[(j * 4 + i) % TILES], a0, a1, a2, a3, pb[0][0], pb[0][1]);
                }
            }
        }
    }

    // the warps' parts: tile (j, i) has values (8j + g) * VN + 2i and the next, heads 2t and 2t + 1
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        if (g == 0) { ms[warp][2 * t + h] = m[h]; ls[warp][2 * t + h] = l[h]; }
    }
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        const int d = (i / (VN / 2) * 8 + g) * VN + i % (VN / 2) * 2;
        *reinterpret_cast<float2 *>(&os[warp][2 * t][d]) = make_float2(o[i][0], o[i][2]);
        *reinterpret_cast<float2 *>(&os[warp][2 * t + 1][d]) = make_float2(o[i][1], o[i][3]);
    }
    __syncthreads();
    const long slot = ((long)row * p.chunks + chunk) * p.q_heads + q_head0;
    for (int i = tid; i < heads * DP; i += WARPS * 32) {
        const int h = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, ms[w][h]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = exp2f(ms[w][h] - ref);
            sum += f * ls[w][h];
            v += f * os[w][h][d];
        }
        if (p.chunks == 1) {
            if (d < dim) dt<T>::st((T *)p.y + (long)row * p.y_ld + (long)(q_head0 + h) * dim + d, sum == 0.f ? 0.f : v / sum);
            if (d == 0 && p.lse) p.lse[(long)row * p.q_heads + q_head0 + h] = sum == 0.f ? -INFINITY : (top - SHIFT<T>) * LN2 + logf(sum);
        } else {
            if (d < dim) p.part[(slot + h) * (dim + 2) + 2 + d] = v;
            if (d == 0) {
                p.part[(slot + h) * (dim + 2)] = top;
                p.part[(slot + h) * (dim + 2) + 1] = sum;
            }
        }
    }
}

// the chunks of a row and head, joined
template <typename T> __global__ void __launch_bounds__(256) paged_join_kernel(AttnParams p)
{
    pdl_enter();
    const int row = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads, dim = p.c.dim;
    int first, last;
    positions(p, row, first, last);
    if (last < first) return;
    const int used = (last - first + p.chunk - 1) / p.chunk;
    const float *part = p.part + ((long)row * p.chunks * p.q_heads + head) * (dim + 2);
    const long step = (long)p.q_heads * (dim + 2);
    float top = -INFINITY;
    for (int c = 0; c < used; c++) top = fmaxf(top, part[c * step]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int d = threadIdx.x; d < dim; d += blockDim.x) {
        float sum = 0.f, v = 0.f;
        for (int c = 0; c < used; c++) {
            const float f = exp2f(part[c * step] - ref);
            sum += f * part[c * step + 1];
            v += f * part[c * step + 2 + d];
        }
        dt<T>::st((T *)p.y + (long)row * p.y_ld + (long)head * dim + d, sum == 0.f ? 0.f : v / sum);
        if (d == 0 && p.lse) p.lse[(long)row * p.q_heads + head] = sum == 0.f ? -INFINITY : (top - SHIFT<T>) * LN2 + logf(sum);
    }
}

template <typename T> int launch_attn(const AttnParams &p, cudaStream_t st)
{
    const dim3 grid((unsigned)(p.rows * p.chunks), (unsigned)(p.c.heads * p.head_tiles));
    if (p.c.dim <= 64) thb_launch(paged_attn_kernel<T, 64>, grid, WARPS * 32, st, p);
    else if (p.c.dim <= 128) thb_launch(paged_attn_kernel<T, 128>, grid, WARPS * 32, st, p);
    else thb_launch(paged_attn_kernel<T, 256>, grid, WARPS * 32, st, p);
    const int rc = THB_LAUNCH_CHECK("paged_attn_kernel");
    if (rc || p.chunks == 1) return rc;
    thb_launch(paged_join_kernel<T>, (unsigned)(p.rows * p.q_heads), (unsigned)((p.c.dim + 31) / 32 * 32), st, p);
    return THB_LAUNCH_CHECK("paged_join_kernel");
}

// tokens a CTA, and how many CTAs share the longest row: four CTAs to each of a B200's 148 SMs where the rows are max_len long
void split(const thb_paged_attn_desc *d, int *chunk, int *chunks)
{
    const long share = d->q_heads / d->cache.heads, base = (long)d->rows * d->cache.heads * ((share + 7) / 8);
    const long span = d->window && d->window < d->max_len ? d->window : d->max_len;
    const long want = (4 * 148 + base - 1) / base;
    long c = (span + want - 1) / want;
    c = (c + 63) / 64 * 64;
    *chunk = (int)(c < 64 ? 64 : c > 2048 ? 2048 : c);
    *chunks = (int)((span + *chunk - 1) / *chunk);
    if (*chunks < 1) *chunks = 1;
}

const char *attn_fault(const thb_paged_attn_desc *d)
{
    const int al = thb_channel_align(d->cache.dtype);
    const char *why = thb_kv_cache_fault(&d->cache);
    if (why) return why;
    if (d->q_heads < 1 || d->q_heads % d->cache.heads) return "thb_paged_attn_fwd: q_heads is below 1 or no multiple of the cache's heads";
    if (d->max_len < 0 || d->window < 0) return "thb_paged_attn_fwd: max_len or window is negative";
    if (d->max_len > 1 << 30) return "thb_paged_attn_fwd: max_len above 2^30";
    if (!(fabsf(d->scale) < INFINITY)) return "thb_paged_attn_fwd: scale is not finite";
    if (!d->len) return "thb_paged_attn_fwd: len must be set";
    if (!d->seq && d->rows > d->cache.sequences) return "thb_paged_attn_fwd: more rows than sequences, and no seq";
    const long w = (long)d->q_heads * d->cache.dim;
    if (d->q_ld < w || d->y_ld < w || d->q_ld % al || d->y_ld % al) return "thb_paged_attn_fwd: q_ld or y_ld is below the row or no multiple of the alignment";
    return nullptr;
}

}  // namespace

extern "C" size_t thb_paged_attn_scratch(const thb_paged_attn_desc *d)
{
    if (!d || d->rows < 1 || d->cache.heads < 1 || d->q_heads < 1 || d->max_len < 0 || d->window < 0 || d->cache.dim < 1) return 0;
    int chunk, chunks;
    split(d, &chunk, &chunks);
    return chunks == 1 ? 0 : (size_t)d->rows * chunks * d->q_heads * (d->cache.dim + 2) * sizeof(float);
}

extern "C" int thb_paged_attn_fwd(const thb_paged_attn_desc *d, const void *q, void *y, thb_stream s)
{
    if (!d) return THB_ERR_ARG;
    const int dtype = d->cache.dtype;
    if (dtype != THB_F32 && dtype != THB_F16 && dtype != THB_BF16)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_paged_attn_fwd: dtype is not THB_F32, THB_F16 or THB_BF16");
    if (d->rows < 0) return thb_refuse(THB_ERR_ARG, "thb_paged_attn_fwd: rows < 0");
    if (d->rows == 0) return THB_OK;
    const char *why = attn_fault(d);
    if (why) return thb_refuse(THB_ERR_ARG, why);
    if (!q || !y || thb_misaligned(q) || thb_misaligned(y)) return thb_refuse(THB_ERR_ARG, "thb_paged_attn_fwd: q or y is missing or not 16-byte aligned");
    AttnParams p = {d->cache, d->len, d->seq, q, y, d->lse, (float *)d->scratch, d->rows, d->q_heads, d->q_ld, d->y_ld, d->max_len, d->window,
                    d->q_heads / d->cache.heads, 0, 0, 0, d->scale};
    p.head_tiles = (p.share + 7) / 8;
    split(d, &p.chunk, &p.chunks);
    if ((long)p.rows * p.chunks >= 1L << 31 || (long)p.rows * p.q_heads >= 1L << 31 || (long)p.c.heads * p.head_tiles > 65535)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_paged_attn_fwd: more rows, chunks or heads than a launch has blocks");
    if (d->scratch_bytes < thb_paged_attn_scratch(d) || (p.chunks > 1 && (!d->scratch || (reinterpret_cast<uintptr_t>(d->scratch) & 3))))
        return thb_refuse(THB_ERR_ARG, "thb_paged_attn_fwd: scratch is missing, misaligned or smaller than thb_paged_attn_scratch says");
    switch (dtype) {
    case THB_F32: return launch_attn<float>(p, (cudaStream_t)s);
    case THB_F16: return launch_attn<__half>(p, (cudaStream_t)s);
    default: return launch_attn<__nv_bfloat16>(p, (cudaStream_t)s);
    }
}
