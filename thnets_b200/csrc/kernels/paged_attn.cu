// Attention of one new token a sequence over a paged cache: y_h = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q_h.k_j - max), over the
// positions j of [max(0, len - window), len).
// HBM-bound on the cache: 4 * heads / kv_heads operations for every 2 values read.  One pass with a running maximum and sum; both
// products run on the tensor cores (mma.sync m16n8k16: 16 tokens or 16 values of a head by the 8 query heads that share a key
// head; tcgen05's 128-row tiles would be mostly empty).  Each warp walks tiles of 16 tokens, which come through a ring of its own in
// shared memory by cp.async of 16 bytes: what is under way does not wait for what is multiplied, and no warp for another.
//   S^T[16 tokens][8 heads] = K Q^T:   K by ldmatrix as it lies; lane (g = lane / 4, t = lane % 4) gets tokens g and g + 8, heads 2t and 2t + 1.
//   O^T[16 values][8 heads] = V^T P^T: V by transposing ldmatrix, P by a transposing move.
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
__device__ __forceinline__ uint4 ldmatrix4(uint32_t at)
{
    uint4 v;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ldmatrix4_trans(uint32_t at)
{
    uint4 v;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
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

// Shared memory: a warp's ring of STAGES tiles, 16 tokens' keys and then their values.  Tiles of 4 and 8 KB leave room for four and two CTAs
// of four warps on an SM, larger ones for one.
template <typename T, int DP> struct Shape {
    static constexpr int ROW = DP * (int)sizeof(T), HALF = 16 * ROW, TILE = 2 * HALF;
    static constexpr int WARPS = TILE <= 8192 ? 4 : TILE == 16384 ? 6 : 3, STAGES = TILE <= 8192 ? 3 : 2;
    static constexpr int PIECES = ROW / 16;                                     // 16-byte pieces of a row
    static constexpr int QWORDS = sizeof(T) == 4 ? DP * 12 : DP * 4;            // words of Q in operand order
    static constexpr int RING = WARPS * STAGES * TILE, SMEM = RING + QWORDS * 4 + WARPS * 64;
    static constexpr int CTAS = TILE <= 4096 ? 4 : TILE <= 8192 ? 2 : 1;
};

template <typename T, int DP>
__global__ void __launch_bounds__(Shape<T, DP>::WARPS * 32, Shape<T, DP>::CTAS) paged_attn_kernel(AttnParams p)
{
    using S = Shape<T, DP>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int WARPS = S::WARPS, STAGES = S::STAGES, VN = Vec16<T>::N, PIECES = S::PIECES, ROW = S::ROW;
    constexpr int TILES = DP / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    uint32_t *const qs = reinterpret_cast<uint32_t *>(smem + S::RING);
    float *const ms = reinterpret_cast<float *>(smem + S::RING + S::QWORDS * 4), *const ls = ms + WARPS * 8;
    pdl_enter();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, dim = p.c.dim;
    // heads of a chunk are neighbours in the grid: a token's keys of all heads lie side by side
    const int head_blocks = p.c.heads * p.head_tiles, hb = blockIdx.x % head_blocks, rc = blockIdx.x / head_blocks;
    const int row = rc / p.chunks, chunk = rc % p.chunks;
    const int kv_head = hb / p.head_tiles, head0 = hb % p.head_tiles * 8, heads = min(8, p.share - head0);
    const int q_head0 = kv_head * p.share + head0;
    int first, last;
    positions(p, row, first, last);
    if (last < first) return;
    // tiles begin at multiples of 16, so that one lies in one page where pages are multiples of 16 tokens
    const int origin = first & ~15, begin = origin + chunk * p.chunk, end = min(last, begin + p.chunk);
    if (begin >= last && (chunk > 0 || p.chunks > 1)) return;

    const int seq = p.seq ? p.seq[row] : row;
    const int *table = p.c.table + (long)((unsigned)seq < (unsigned)p.c.sequences ? seq : 0) * p.c.table_ld;
    const bool whole = p.c.page_len % 16 == 0;
    const uint32_t ring = smem_u32(smem) + warp * STAGES * S::TILE;
    const long head_at = kv_head * p.c.head_stride;

    // pieces of a row, permuted so that the operands' loads meet no bank twice: 16-bit rows by ldmatrix of 8 rows; fp32 keys 4 pieces of 2
    // rows, values 2 pieces of every other of 8 rows
    auto key_piece = [](int r, int c) { return r * ROW + ((c ^ (F32 ? (r & 1) << 2 : r & 7)) << 4); };
    auto value_piece = [](int r, int c) { return r * ROW + ((c ^ (F32 ? (r >> 1 & 3) << 1 : r & 7)) << 4); };

    // ---- a tile's loads.  Its page is looked up a tile earlier: one for all of it, or one a token (lane) where tiles cross pages
    auto page_of = [&](int tile) {
        const int token = whole ? tile : tile + (lane & 15);
        return token < end ? __ldg(table + token / p.c.page_len) : 0;
    };
    int ftile = begin + warp * 16, fslot = 0, fpage = page_of(ftile);
    uint32_t seen[STAGES];  // tokens that count, of the tiles under way
    auto fetch = [&](uint32_t &mask) {
        mask = 0;
        if (ftile < end) {
            const int token = ftile + (lane & 15);
            const bool there = (unsigned)fpage < (unsigned)p.c.pages, ok = there && token >= first && token < end;
            if (!there && token >= first && token < end) *p.c.status = THB_ERR_ARG;
            mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            const long mine = ok ? fpage * p.c.page_stride + (token % p.c.page_len) * p.c.token_stride + head_at : 0;
            const uint32_t to = ring + fslot * S::TILE;
            constexpr int RS = PIECES >= 32 ? 1 : 32 / PIECES;  // rows a warp's instruction covers
#pragma unroll
            for (int i = 0; i < 16; i += RS)
#pragma unroll
                for (int h = 0; h < (PIECES > 32 ? PIECES / 32 : 1); h++) {
                    const int r = i + lane / PIECES % RS, c = h * 32 + lane % PIECES;
                    const long at = __shfl_sync(0xffffffffu, mine, r);
                    const bool in = (mask >> r & 1) && c * VN < dim;
                    const long o = in ? at + c * VN : 0;
                    cp_async16(to + key_piece(r, c), (const T *)p.c.k + o, in ? 16 : 0);
                    cp_async16(to + S::HALF + value_piece(r, c), (const T *)p.c.v + o, in ? 16 : 0);
                }
            ftile += WARPS * 16;
            fpage = page_of(ftile);
        }
        cp_async_commit();
        fslot = fslot + 1 == STAGES ? 0 : fslot + 1;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(seen[i]);

    // Q in operand order: head g's values that a lane's B registers take beside each piece of the keys
    for (int j = warp; j < DP / 16; j += WARPS) {
        const T *from = (const T *)p.q + (long)row * p.q_ld + (long)(q_head0 + (g < heads ? g : 0)) * dim;
        if constexpr (F32) {
            const int d = 16 * j + 4 * t;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (g < heads && d < dim) v = *reinterpret_cast<const uint4 *>(from + d);
            uint32_t a[4][3];
            parts_of(v.x, a[0]); parts_of(v.y, a[1]); parts_of(v.z, a[2]); parts_of(v.w, a[3]);
#pragma unroll
            for (int i = 0; i < 3; i++) {
                qs[(j * 6 + 2 * i) * 32 + lane] = tops(a[0][i], a[1][i]);
                qs[(j * 6 + 2 * i + 1) * 32 + lane] = tops(a[2][i], a[3][i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int d = 16 * j + 8 * i + 2 * t;
                qs[(j * 2 + i) * 32 + lane] = g < heads && d < dim ? *reinterpret_cast<const uint32_t *>(from + d) : 0u;
            }
        }
    }
    __syncthreads();

    float o[TILES][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < TILES; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) o[i][k] = 0.f;
    const float scale = p.scale * LOG2E;
    // this lane's rows and pieces for ldmatrix: keys [tokens 0-7, 8-15][values 0-7, 8-15] of 16 values, values the other way round
    const uint32_t key_at = key_piece((lane & 7) + (lane >> 3 & 1) * 8, lane >> 4), value_at = value_piece((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);

    int slot = 0;
    for (int tile = begin + warp * 16; tile < end; tile += WARPS * 16) {
        __syncwarp();  // (all lanes have read the tile whose place is loaded next)
        fetch(seen[STAGES - 1]);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t at = ring + slot * S::TILE, mask = seen[0];
#pragma unroll
        for (int i = 0; i + 1 < STAGES; i++) seen[i] = seen[i + 1];
        const uint8_t *const mem = smem + warp * STAGES * S::TILE + slot * S::TILE;
        slot = slot + 1 == STAGES ? 0 : slot + 1;

        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < DP / 16; j++) {
            if constexpr (F32) {
                const uint4 a = *reinterpret_cast<const uint4 *>(mem + key_piece(g, j * 4 + t)), b = *reinterpret_cast<const uint4 *>(mem + key_piece(g + 8, j * 4 + t));
                uint32_t x[4][3], y[4][3];
                parts_of(a.x, x[0]); parts_of(a.y, x[1]); parts_of(a.z, x[2]); parts_of(a.w, x[3]);
                parts_of(b.x, y[0]); parts_of(b.y, y[1]); parts_of(b.z, y[2]); parts_of(b.w, y[3]);
                float c[4] = {0.f, 0.f, 0.f, 0.f};  // (the tensor core truncates its sums: 16 values at a time, added in fp32)
#pragma unroll
                for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                    for (int i = sum; i >= 0; i--)
                        mma<T>(c, tops(x[0][i], x[1][i]), tops(y[0][i], y[1][i]), tops(x[2][i], x[3][i]), tops(y[2][i], y[3][i]),
                               qs[(j * 6 + 2 * (sum - i)) * 32 + lane], qs[(j * 6 + 2 * (sum - i) + 1) * 32 + lane]);
#pragma unroll
                for (int i = 0; i < 4; i++) s[i] += c[i];
            } else {
                const uint4 a = ldmatrix4(at + (key_at ^ (j & 3) * 32) + (j >> 2) * 128);
                mma<T>(s, a.x, a.y, a.z, a.w, qs[j * 64 + lane], qs[j * 64 + 32 + lane]);
            }
        }
        // the softmax's running maximum and sum of heads 2t and 2t + 1; a lane has tokens g and g + 8 of the sum
        const bool see0 = mask >> g & 1, see1 = mask >> (g + 8) & 1;
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
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < DP / 32; j++) {
                // tokens 2t, 2t + 1, 2t + 8 and 2t + 9, values (8j + g) * 4 and the next three
                uint32_t w[4][4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(mem + S::HALF + value_piece(2 * t + (r & 1) + 8 * (r >> 1), j * 8 + g));
                    w[r][0] = v.x; w[r][1] = v.y; w[r][2] = v.z; w[r][3] = v.w;
                }
#pragma unroll
                for (int i = 0; i < 2; i++) {  // values 2i and 2i + 1 of the piece
                    uint32_t x[4][2][3];
#pragma unroll
                    for (int r = 0; r < 4; r++) { parts_of(w[r][2 * i], x[r][0]); parts_of(w[r][2 * i + 1], x[r][1]); }
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int sum = 2; sum >= 0; sum--)
#pragma unroll
                        for (int a = sum; a >= 0; a--)
                            mma<T>(c, tops(x[0][0][a], x[1][0][a]), tops(x[0][1][a], x[1][1][a]), tops(x[2][0][a], x[3][0][a]),
                                   tops(x[2][1][a], x[3][1][a]), pb[(sum - a) % PP][0], pb[(sum - a) % PP][1]);
#pragma unroll
                    for (int k = 0; k < 4; k++) o[j * 2 + i][k] += c[k];
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const uint4 a = ldmatrix4_trans(at + S::HALF + (value_at ^ (i & 3) * 32) + (i >> 2) * 128);
                mma<T>(o[i], a.x, a.y, a.z, a.w, pb[1][0], pb[1][1]);
                mma<T>(o[i], a.x, a.y, a.z, a.w, pb[0][0], pb[0][1]);
            }
        }
    }
    cp_async_wait<0>();
    __syncwarp();

    // The warps' parts, each in its own ring.  o[i]: heads 2t and 2t + 1 of two values: 16i + g and 16i + g + 8, or in fp32 those of piece
    // 8 (i / 2) + g, 2 (i % 2) and the next.
    float *const mine = reinterpret_cast<float *>(smem + warp * STAGES * S::TILE);
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        if (g == 0) { ms[warp * 8 + 2 * t + h] = m[h]; ls[warp * 8 + 2 * t + h] = l[h]; }
    }
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        const int d0 = F32 ? (i / 2 * 8 + g) * 4 + i % 2 * 2 : 16 * i + g, d1 = F32 ? d0 + 1 : d0 + 8;
        mine[2 * t * DP + d0] = o[i][0];
        mine[(2 * t + 1) * DP + d0] = o[i][1];
        mine[2 * t * DP + d1] = o[i][2];
        mine[(2 * t + 1) * DP + d1] = o[i][3];
    }
    __syncthreads();
    const long slot_at = ((long)row * p.chunks + chunk) * p.q_heads + q_head0;
    for (int i = tid; i < heads * DP; i += WARPS * 32) {
        const int h = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, ms[w * 8 + h]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = exp2f(ms[w * 8 + h] - ref);
            sum += f * ls[w * 8 + h];
            v += f * reinterpret_cast<const float *>(smem + w * STAGES * S::TILE)[h * DP + d];
        }
        if (p.chunks == 1) {
            if (d < dim) dt<T>::st((T *)p.y + (long)row * p.y_ld + (long)(q_head0 + h) * dim + d, sum == 0.f ? 0.f : v / sum);
            if (d == 0 && p.lse) p.lse[(long)row * p.q_heads + q_head0 + h] = sum == 0.f ? -INFINITY : (top - SHIFT<T>) * LN2 + logf(sum);
        } else {
            if (d < dim) p.part[(slot_at + h) * dim + d] = v;
            if (d == 0) reinterpret_cast<float2 *>(p.part + (long)p.rows * p.chunks * p.q_heads * dim)[slot_at + h] = make_float2(top, sum);
        }
    }
}

// The chunks of a row and head, joined: four warps take every fourth chunk, a lane four or eight values of it.
template <typename T> __global__ void __launch_bounds__(128) paged_join_kernel(AttnParams p)
{
    __shared__ float sums[4], vs[4][256];
    pdl_enter();
    const int row = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads, dim = p.c.dim, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int first, last;
    positions(p, row, first, last);
    if (last < first) return;
    const int used = (last - (first & ~15) + p.chunk - 1) / p.chunk;
    const long slot = (long)row * p.chunks * p.q_heads + head;
    const float *const part = p.part + slot * dim;
    const float2 *const stats = reinterpret_cast<const float2 *>(p.part + (long)p.rows * p.chunks * p.q_heads * dim) + slot;
    const int d = lane * 4;
    // (every warp needs the largest of all chunks)
    float top = -INFINITY;
    for (int c = lane; c < used; c += 32) top = fmaxf(top, stats[(long)c * p.q_heads].x);
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 8
    for (int c = warp; c < used; c += 4) {
        const float2 s = stats[(long)c * p.q_heads];
        const float *const v = part + (long)c * p.q_heads * dim;
        const float f = exp2f(s.x - ref);
        sum += f * s.y;
        if (d < dim) {
            const float4 w = *reinterpret_cast<const float4 *>(v + d);
            a.x += f * w.x; a.y += f * w.y; a.z += f * w.z; a.w += f * w.w;
        }
        if (d + 128 < dim) {
            const float4 w = *reinterpret_cast<const float4 *>(v + d + 128);
            b.x += f * w.x; b.y += f * w.y; b.z += f * w.z; b.w += f * w.w;
        }
    }
    *reinterpret_cast<float4 *>(&vs[warp][d]) = a;
    *reinterpret_cast<float4 *>(&vs[warp][d + 128]) = b;
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    for (int i = threadIdx.x; i < dim; i += 128) {
        const float v = (vs[0][i] + vs[1][i]) + (vs[2][i] + vs[3][i]);
        dt<T>::st((T *)p.y + (long)row * p.y_ld + (long)head * dim + i, sum == 0.f ? 0.f : v / sum);
    }
    if (threadIdx.x == 0 && p.lse) p.lse[(long)row * p.q_heads + head] = sum == 0.f ? -INFINITY : (top - SHIFT<T>) * LN2 + logf(sum);
}

template <typename T, int DP> int launch_heads(const AttnParams &p, cudaStream_t st)
{
    using S = Shape<T, DP>;
    const auto kern = paged_attn_kernel<T, DP>;
    static bool set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e != cudaSuccess) return thb_note_launch(e, "paged_attn_kernel attributes");
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)p.rows * p.chunks * p.c.heads * p.head_tiles));
    cfg.blockDim = dim3(S::WARPS * 32);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = thb_pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    return thb_note_launch(e != cudaSuccess ? e : cudaGetLastError(), "paged_attn_kernel");
}

template <typename T> int launch_attn(const AttnParams &p, cudaStream_t st)
{
    const int rc = p.c.dim <= 64 ? launch_heads<T, 64>(p, st) : p.c.dim <= 128 ? launch_heads<T, 128>(p, st) : launch_heads<T, 256>(p, st);
    if (rc || p.chunks == 1) return rc;
    thb_launch(paged_join_kernel<T>, (unsigned)(p.rows * p.q_heads), 128, st, p);
    return THB_LAUNCH_CHECK("paged_join_kernel");
}

// tokens a CTA, and how many CTAs share the longest row: four CTAs to each of a B200's 148 SMs where the rows are max_len long
void split(const thb_paged_attn_desc *d, int *chunk, int *chunks)
{
    const long share = d->q_heads / d->cache.heads, base = (long)d->rows * d->cache.heads * ((share + 7) / 8);
    const long span = d->window && d->window < d->max_len ? d->window + 15L : d->max_len;  // (from a multiple of 16 on)
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
    if ((double)p.rows * p.chunks * p.c.heads * p.head_tiles >= 2147483648.0 || (long)p.rows * p.q_heads >= 1L << 31)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_paged_attn_fwd: more rows, chunks or heads than a launch has blocks");
    if (d->scratch_bytes < thb_paged_attn_scratch(d) || (p.chunks > 1 && (!d->scratch || thb_misaligned(d->scratch))))
        return thb_refuse(THB_ERR_ARG, "thb_paged_attn_fwd: scratch is missing, misaligned or smaller than thb_paged_attn_scratch says");
    switch (dtype) {
    case THB_F32: return launch_attn<float>(p, (cudaStream_t)s);
    case THB_F16: return launch_attn<__half>(p, (cudaStream_t)s);
    default: return launch_attn<__nv_bfloat16>(p, (cudaStream_t)s);
    }
}
