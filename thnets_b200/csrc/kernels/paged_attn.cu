// Attention of one new token a sequence over a paged cache: y_h = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q_h.k_j - max), over the
// positions j of [max(0, len - window), len).
// HBM-bound on the cache: 4 * heads / kv_heads operations for every 2 values read.  One pass with a running maximum and sum; both
// products run on the tensor cores (mma.sync m16n8k16: 16 tokens or 16 values of a head by the 8 query heads that share a key
// head; tcgen05's 128-row tiles would be mostly empty).  Each warp walks tiles of 16 tokens, which come through a ring of its own in
// shared memory by cp.async of 16 bytes: what is under way does not wait for what is multiplied, and no warp for another.
//   S^T[16 tokens][8 heads] = K Q^T:   K by ldmatrix as it lies; lane (g = lane / 4, t = lane % 4) gets tokens g and g + 8, heads 2t and 2t + 1.
//   O^T[16 values][8 heads] = V^T P^T: V by transposing ldmatrix, P by a transposing move.
// 16-bit types: p is two parts (its nearest value and what is left), so that its rounding does not show.  fp32: chains of FFMA, which take
// fewer instructions than splitting k and v into parts for the tensor cores would.
// The length is split among CTAs by `chunk` tokens.  Up to sixteen are a cluster and join their parts through distributed shared memory; more
// leave them to a second launch.
#include "tokens.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace {

struct AttnParams {
    thb_kv_cache c;
    const int *len, *seq;
    const void *q;
    void *y;
    float *lse, *part;
    int rows, q_heads, q_ld, y_ld, max_len, window, share, head_tiles, chunk, chunks, cluster;
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
__device__ __forceinline__ float exp2_of(float x)  // 2^-22 off at most; results below 2^-126 are zero
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// of four warps on an SM, of 16 and 32 KB for two and one of three.  HT: query heads a CTA takes at most.
template <typename T, int DP, int HT> struct Shape {
    static constexpr int ROW = (DP * (int)sizeof(T) + 127) / 128 * 128, HALF = 16 * ROW, TILE = 2 * HALF;
    static constexpr int WARPS = TILE <= 8192 ? 4 : 3, STAGES = TILE <= 12288 ? 3 : 2;
    static constexpr int PIECES = DP * (int)sizeof(T) / 16;                                    // 16-byte pieces of a row
    static constexpr int QWORDS = sizeof(T) == 4 ? HT * DP : 0;                                // words of Q, where they are not in registers
    // and the warps' maxima and sums, the CTA's, and the warps' p in fp32
    static constexpr int RING = WARPS * STAGES * TILE, SMEM = RING + QWORDS * 4 + (WARPS + 1) * HT * 8 + (sizeof(T) == 4 ? WARPS * HT * 64 : 0);
    static constexpr int CTAS = TILE <= 4096 ? 4 : TILE <= 16384 ? 2 : 1;
};

template <typename T, int DP, int HT>
__global__ void __launch_bounds__(Shape<T, DP, HT>::WARPS * 32, Shape<T, DP, HT>::CTAS) paged_attn_kernel(AttnParams p)
{
    using S = Shape<T, DP, HT>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int WARPS = S::WARPS, STAGES = S::STAGES, VN = Vec16<T>::N, PIECES = S::PIECES, ROW = S::ROW;
    extern __shared__ __align__(128) uint8_t smem[];
    float *const qs = reinterpret_cast<float *>(smem + S::RING), *const ms = qs + S::QWORDS, *const ls = ms + WARPS * HT, *const joined = ls + WARPS * HT;
    pdl_enter();

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, dim = p.c.dim;
    // heads of a chunk are neighbours in the grid: a token's keys of all heads lie side by side
    const int row = blockIdx.z, chunk = blockIdx.y, kv_head = blockIdx.x / p.head_tiles;
    const int head0 = blockIdx.x % p.head_tiles * HT, heads = min(HT, p.share - head0);
    const int q_head0 = kv_head * p.share + head0;
    // (where no window moves the chunks the first page is asked for together with the length)
    const int seq = p.seq ? p.seq[row] : row;
    const int *table = p.c.table + (long)((unsigned)seq < (unsigned)p.c.sequences ? seq : 0) * p.c.table_ld;
    const bool whole = p.c.page_len % 16 == 0;
    const long start = (long)chunk * p.chunk + warp * 16 + (whole ? 0 : lane & 15);
    int fpage = !p.window && start < (long)p.c.table_ld * p.c.page_len ? table[(int)start / p.c.page_len] : 0;
    int first, last;
    positions(p, row, first, last);
    if (last < first) return;
    // tiles begin at multiples of 16, so that one lies in one page where pages are multiples of 16 tokens
    const int origin = first & ~15, begin = origin + chunk * p.chunk, end = min(last, begin + p.chunk);
    if (begin >= last && (chunk > 0 || (p.chunks > 1 && !p.cluster))) return;  // (an empty row's zeros: by the first CTA, or by the join)
    const uint32_t ring = smem_u32(smem) + warp * STAGES * S::TILE;
    const long head_at = kv_head * p.c.head_stride;

    // pieces of a row, permuted so that the loads meet no bank twice: 16-bit rows by ldmatrix of 8 rows; fp32 keys 2 pieces of 4 rows (fp32
    // values whole rows)
    auto key_piece = [](int r, int c) { return r * ROW + ((c ^ (F32 ? (r & 3) << 1 : r & 7)) << 4); };
    auto value_piece = [](int r, int c) { return r * ROW + ((c ^ (F32 ? 0 : r & 7)) << 4); };

    // ---- a tile's loads.  Its page is looked up a tile earlier: one for all of it, or one a token (lane) where tiles cross pages
    auto page_of = [&](int tile) {
        const int token = whole ? tile : tile + (lane & 15);
        return token < end ? table[token / p.c.page_len] : 0;
    };
    constexpr int COPIES = PIECES / 2;  // of 32 pieces
    auto row_of = [&](int i) { return (i * 32 + lane) / PIECES; };
    auto piece_of = [&](int i) { return (i * 32 + lane) % PIECES; };
    int ftile = begin + warp * 16, fslot = 0;
    if (p.window) fpage = page_of(ftile);
    uint32_t seen[STAGES];  // tokens that count, of the tiles under way
    auto fetch = [&](uint32_t &mask) {
        mask = 0;
        if (ftile < end) {
            const uint32_t to = ring + fslot * S::TILE;
            if (whole && ftile >= first && ftile + 16 <= end && (unsigned)fpage < (unsigned)p.c.pages) {
                mask = 0xffffu;
                const long at = fpage * p.c.page_stride + ftile % p.c.page_len * p.c.token_stride + head_at;
#pragma unroll
                for (int i = 0; i < COPIES; i++) {
                    const int r = row_of(i), c = piece_of(i);
                    const long o = c * VN < dim ? at + r * p.c.token_stride + c * VN : 0;
                    const uint32_t size = c * VN < dim ? 16 : 0;
                    cp_async16(to + key_piece(r, c), (const T *)p.c.k + o, size);
                    cp_async16(to + S::HALF + value_piece(r, c), (const T *)p.c.v + o, size);
                }
            } else {
                const int token = ftile + (lane & 15);
                const bool there = (unsigned)fpage < (unsigned)p.c.pages, counts = token >= first && token < end, ok = there && counts;
                if (!there && counts) *p.c.status = THB_ERR_ARG;
                mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                const long mine = ok ? fpage * p.c.page_stride + (token % p.c.page_len) * p.c.token_stride + head_at : 0;
#pragma unroll
                for (int i = 0; i < COPIES; i++) {
                    const int r = row_of(i), c = piece_of(i);
                    const long at = __shfl_sync(0xffffffffu, mine, r);
                    const bool in = (mask >> r & 1) && c * VN < dim;
                    const long o = in ? at + c * VN : 0;
                    cp_async16(to + key_piece(r, c), (const T *)p.c.k + o, in ? 16 : 0);
                    cp_async16(to + S::HALF + value_piece(r, c), (const T *)p.c.v + o, in ? 16 : 0);
                }
            }
            ftile += WARPS * 16;
            fpage = page_of(ftile);
        }
        cp_async_commit();
        fslot = fslot + 1 == STAGES ? 0 : fslot + 1;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(seen[i]);

    // Q: in 16 bits as the B operands beside each piece of the keys, in registers: head 8n + g's values; in fp32 as rows in shared memory
    constexpr int NT = (HT + 7) / 8;
    uint32_t qb[F32 ? 1 : DP / 16][NT][2];
    if constexpr (F32) {
        for (int i = tid; i < HT * DP; i += WARPS * 32) {
            const int h = i / DP, d = i % DP;
            qs[i] = h < heads && d < dim ? ((const float *)p.q)[(long)row * p.q_ld + (long)(q_head0 + h) * dim + d] : 0.f;
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int j = 0; j < DP / 16; j++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 16 * j + 8 * i + 2 * t, h = 8 * n + g;
                    qb[j][n][i] = h < heads && d < dim ? *reinterpret_cast<const uint32_t *>((const T *)p.q + (long)row * p.q_ld + (long)(q_head0 + h) * dim + d) : 0u;
                }
    }

    const float scale = p.scale * LOG2E;
    int slot = 0;
    // the next tile that is there: its place in shared memory, its tokens that count
    auto next_tile = [&](uint32_t &mask) {
        __syncwarp();  // (all lanes have read the tile whose place is loaded next)
        fetch(seen[STAGES - 1]);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        mask = seen[0];
#pragma unroll
        for (int i = 0; i + 1 < STAGES; i++) seen[i] = seen[i + 1];
        const int at = slot * S::TILE;
        slot = slot + 1 == STAGES ? 0 : slot + 1;
        return at;
    };
    float *const mine = reinterpret_cast<float *>(smem + warp * STAGES * S::TILE);  // (a warp's ring; its part of the result when that is done)

    if constexpr (F32) {
        // lane: half of a token's products (pieces of one parity), then VL tokens' share of 4 values a piece
        constexpr int VP = PIECES > 32 ? 2 : 1, VL = PIECES > 16 ? 1 : 2;
        float o[HT][VP][4], m[HT], l[HT];
#pragma unroll
        for (int h = 0; h < HT; h++) {
            m[h] = -INFINITY;
            l[h] = 0.f;
#pragma unroll
            for (int i = 0; i < VP; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[h][i][k] = 0.f;
        }
        float *const ps = joined + 2 * HT + warp * HT * 16;  // p of this warp's tile, [HT][16]
        for (int tile = begin + warp * 16; tile < end; tile += WARPS * 16) {
            uint32_t mask;
            const uint8_t *const mem = smem + warp * STAGES * S::TILE + next_tile(mask);
            const int mytoken = lane >> 1;
            float s[HT][2];
#pragma unroll
            for (int h = 0; h < HT; h++) s[h][0] = s[h][1] = 0.f;
#pragma unroll
            for (int j = 0; j < PIECES / 2; j++) {
                const float4 k = *reinterpret_cast<const float4 *>(mem + key_piece(mytoken, 2 * j + (lane & 1)));
#pragma unroll
                for (int h = 0; h < HT; h++) {
                    const float4 q = *reinterpret_cast<const float4 *>(qs + h * DP + (2 * j + (lane & 1)) * 4);
                    s[h][0] = fmaf(k.x, q.x, s[h][0]);
                    s[h][1] = fmaf(k.y, q.y, s[h][1]);
                    s[h][0] = fmaf(k.z, q.z, s[h][0]);
                    s[h][1] = fmaf(k.w, q.w, s[h][1]);
                }
            }
            const bool see = mask >> mytoken & 1;
            float shrink[HT];
#pragma unroll
            for (int h = 0; h < HT; h++) {
                float a = s[h][0] + s[h][1];
                a += __shfl_xor_sync(0xffffffffu, a, 1);
                a = see ? a * scale : -INFINITY;
                float top = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                top = fmaxf(top, m[h]);
                const float ref = top == -INFINITY ? 0.f : top;  // (nothing seen yet: every p is zero)
                shrink[h] = exp2_of(m[h] - ref);
                m[h] = top;
                a = exp2_of(a - ref);
                l[h] = l[h] * shrink[h] + a;
                if (!(lane & 1)) ps[h * 16 + mytoken] = a;
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < HT; h++)
#pragma unroll
                for (int i = 0; i < VP; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) o[h][i][k] *= shrink[h];
#pragma unroll
            for (int i = 0; i < 16; i += VL) {
                const int r = i + (VL > 1 ? lane >> 4 : 0), c = VL > 1 ? lane & 15 : PIECES < 32 && lane >= PIECES ? 0 : lane;
                float4 v[VP];
#pragma unroll
                for (int q = 0; q < VP; q++) v[q] = *reinterpret_cast<const float4 *>(mem + S::HALF + value_piece(r, c + 32 * q));
#pragma unroll
                for (int h = 0; h < HT; h++) {
                    const float w = ps[h * 16 + r];
#pragma unroll
                    for (int q = 0; q < VP; q++) {
                        o[h][q][0] = fmaf(w, v[q].x, o[h][q][0]);
                        o[h][q][1] = fmaf(w, v[q].y, o[h][q][1]);
                        o[h][q][2] = fmaf(w, v[q].z, o[h][q][2]);
                        o[h][q][3] = fmaf(w, v[q].w, o[h][q][3]);
                    }
                }
            }
        }
        cp_async_wait<0>();
        __syncwarp();
#pragma unroll
        for (int h = 0; h < HT; h++) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
            if (lane == 0) { ms[warp * HT + h] = m[h]; ls[warp * HT + h] = l[h]; }
#pragma unroll
            for (int q = 0; q < VP; q++) {
                if (VL > 1)
#pragma unroll
                    for (int k = 0; k < 4; k++) o[h][q][k] += __shfl_xor_sync(0xffffffffu, o[h][q][k], 16);
                if (lane < PIECES)
                    *reinterpret_cast<float4 *>(mine + h * DP + (lane + 32 * q) * 4) = make_float4(o[h][q][0], o[h][q][1], o[h][q][2], o[h][q][3]);
            }
        }
    } else {
        constexpr int TILES = DP / 16;
        const uint32_t ring_at = smem_u32(smem) + warp * STAGES * S::TILE;
        // this lane's rows and pieces for ldmatrix: keys [tokens 0-7, 8-15][values 0-7, 8-15] of 16 values, values the other way round
        const uint32_t key_at = key_piece((lane & 7) + (lane >> 3 & 1) * 8, lane >> 4), value_at = value_piece((lane & 7) + (lane >> 4) * 8, lane >> 3 & 1);
        float o[NT][TILES][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[n][i][k] = 0.f;
        }
        for (int tile = begin + warp * 16; tile < end; tile += WARPS * 16) {
            uint32_t mask;
            const uint32_t at = ring_at + next_tile(mask);
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) s[n][k] = 0.f;
#pragma unroll
            for (int j = 0; j < DP / 16; j++) {
                const uint4 a = ldmatrix4(at + (key_at ^ (j & 3) * 32) + (j >> 2) * 128);
#pragma unroll
                for (int n = 0; n < NT; n++) mma<T>(s[n], a.x, a.y, a.z, a.w, qb[j][n][0], qb[j][n][1]);
            }
            // the softmax's running maximum and sum of heads 8n + 2t and the next; a lane has tokens g and g + 8 of the sum
            const bool see0 = mask >> g & 1, see1 = mask >> (g + 8) & 1;
            uint32_t pb[NT][2][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float pr[4], shrink[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float a = see0 ? s[n][h] * scale : -INFINITY, b = see1 ? s[n][2 + h] * scale : -INFINITY;
                    float top = fmaxf(a, b);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    top = fmaxf(top, m[n][h]);
                    const float ref = top == -INFINITY ? 0.f : top;  // (nothing seen yet: every p is zero)
                    shrink[h] = exp2_of(m[n][h] - ref);
                    m[n][h] = top;
                    pr[h] = exp2_of(a - ref + SHIFT<T>);
                    pr[2 + h] = exp2_of(b - ref + SHIFT<T>);
                    l[n][h] = l[n][h] * shrink[h] + (pr[h] + pr[2 + h]);
                }
                if (__any_sync(0xffffffffu, shrink[0] != 1.f || shrink[1] != 1.f))
#pragma unroll
                    for (int i = 0; i < TILES; i++) {
                        o[n][i][0] *= shrink[0]; o[n][i][1] *= shrink[1]; o[n][i][2] *= shrink[0]; o[n][i][3] *= shrink[1];
                    }
                // p as the B operand: both parts of (token, heads 2t, 2t + 1), transposed to (head, tokens 2t, 2t + 1)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const uint32_t u = pair16<T>(pr[2 * r], pr[2 * r + 1]);
                    const float2 w = wide16<T>(u);
                    pb[n][0][r] = transpose8x8(u);
                    pb[n][1][r] = transpose8x8(pair16<T>(pr[2 * r] - w.x, pr[2 * r + 1] - w.y));
                }
            }
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const uint4 a = ldmatrix4_trans(at + S::HALF + (value_at ^ (i & 3) * 32) + (i >> 2) * 128);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    mma<T>(o[n][i], a.x, a.y, a.z, a.w, pb[n][1][0], pb[n][1][1]);
                    mma<T>(o[n][i], a.x, a.y, a.z, a.w, pb[n][0][0], pb[n][0][1]);
                }
            }
        }
        cp_async_wait<0>();
        __syncwarp();
        // o[n][i]: values 16i + g (twice) and 16i + g + 8, heads 8n + 2t and the next
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 4);
                l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 8);
                l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], 16);
                if (g == 0) { ms[warp * HT + 8 * n + 2 * t + h] = m[n][h]; ls[warp * HT + 8 * n + 2 * t + h] = l[n][h]; }
            }
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) mine[(8 * n + 2 * t + (k & 1)) * DP + 16 * i + g + (k >> 1) * 8] = o[n][i][k];
        }
    }
    __syncthreads();

    // the warps' parts, joined; then the chunks' by the cluster, or by another launch
    const long slot_at = ((long)row * p.chunks + chunk) * p.q_heads + q_head0;
    auto result = [&](int h, int d, float v, float sum, float top) {
        if (d < dim) dt<T>::st((T *)p.y + (long)row * p.y_ld + (long)(q_head0 + h) * dim + d, sum == 0.f ? 0.f : v / sum);
        if (d == 0 && p.lse) p.lse[(long)row * p.q_heads + q_head0 + h] = sum == 0.f ? -INFINITY : (top - SHIFT<T>) * LN2 + logf(sum);
    };
    for (int i = tid; i < heads * DP; i += WARPS * 32) {
        const int h = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) top = fmaxf(top, ms[w * HT + h]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = exp2f(ms[w * HT + h] - ref);
            sum += f * ls[w * HT + h];
            v += f * reinterpret_cast<const float *>(smem + w * STAGES * S::TILE)[i];
        }
        if (p.chunks == 1) result(h, d, v, sum, top);
        else if (p.cluster) {
            reinterpret_cast<float *>(smem)[i] = v;  // (only this thread reads and writes this value of the first warp's part)
            if (d == 0) {
                joined[h] = top;
                joined[HT + h] = sum;
            }
        } else {
            if (d < dim) p.part[(slot_at + h) * dim + d] = v;
            if (d == 0) reinterpret_cast<float2 *>(p.part + (long)p.rows * p.chunks * p.q_heads * dim)[slot_at + h] = make_float2(top, sum);
        }
    }
    if (!p.cluster) return;
    // CTAs without a token have left, and are neither waited for nor read
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    const int used = max(1, (last - origin + p.chunk - 1) / p.chunk);
    for (int i = chunk * (WARPS * 32) + tid; i < heads * DP; i += used * (WARPS * 32)) {
        const int h = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, v = 0.f;
        for (int c = 0; c < used; c++) top = fmaxf(top, *cluster.map_shared_rank(joined + h, c));
        const float ref = top == -INFINITY ? 0.f : top;
        for (int c = 0; c < used; c++) {
            const float f = exp2f(*cluster.map_shared_rank(joined + h, c) - ref);
            sum += f * *cluster.map_shared_rank(joined + HT + h, c);
            v += f * *cluster.map_shared_rank(reinterpret_cast<float *>(smem) + i, c);
        }
        result(h, d, v, sum, top);
    }
    cluster.sync();  // the parts outlive the reads above
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

template <typename T, int DP, int HT> int launch_heads(const AttnParams &p, cudaStream_t st)
{
    using S = Shape<T, DP, HT>;
    const auto kern = paged_attn_kernel<T, DP, HT>;
    static bool set[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return thb_note_launch(e, "paged_attn_kernel attributes");
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.c.heads * p.head_tiles, p.chunks, p.rows);
    cfg.blockDim = dim3(S::WARPS * 32);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (p.cluster) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = attr[n].val.clusterDim.z = 1;
        attr[n].val.clusterDim.y = p.chunks;
        n++;
    }
    if (thb_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    return thb_note_launch(e != cudaSuccess ? e : cudaGetLastError(), "paged_attn_kernel");
}

template <typename T, int DP> int launch_dim(const AttnParams &p, int ht, cudaStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        if (ht == 1) return launch_heads<T, DP, 1>(p, st);
        if (ht == 2) return launch_heads<T, DP, 2>(p, st);
        if (ht == 4) return launch_heads<T, DP, 4>(p, st);
    } else if constexpr (DP <= 128) {
        if (ht == 16) return launch_heads<T, DP, 16>(p, st);
    }
    return launch_heads<T, DP, 8>(p, st);
}

template <typename T> int launch_attn(const AttnParams &p, int ht, cudaStream_t st)
{
    const int rc = p.c.dim <= 64 ? launch_dim<T, 64>(p, ht, st) : p.c.dim <= 96 ? launch_dim<T, 96>(p, ht, st) : p.c.dim <= 128 ? launch_dim<T, 128>(p, ht, st) : launch_dim<T, 256>(p, ht, st);
    if (rc || p.chunks == 1 || p.cluster) return rc;
    thb_launch(paged_join_kernel<T>, (unsigned)(p.rows * p.q_heads), 128, st, p);
    return THB_LAUNCH_CHECK("paged_join_kernel");
}

// How a call is cut: `ht` query heads a CTA at most, `chunk` tokens a CTA, `chunks` CTAs for the longest row, in a cluster or not.
struct Cut {
    int ht, head_tiles, chunk, chunks, cluster;
};
Cut cut_of(const thb_paged_attn_desc *d)
{
    Cut c;
    const int share = d->q_heads / d->cache.heads;
    c.ht = d->cache.dtype == THB_F32 ? (share > 4 ? 8 : share > 2 ? 4 : share) : share > 8 && d->cache.dim <= 128 ? 16 : 8;
    c.head_tiles = (share + c.ht - 1) / c.ht;
    // One wave of CTAs on a B200's 148 SMs (a constant: the size of scratch and the bits of the results do not depend on the device that is current;
    // as many CTAs to each SM as Shape says) where the rows are max_len long; a tile for each of four warps at
    // least.  Of several rows a CTA takes 2048 tokens at most, so that a few long ones among short ones are still many CTAs.
    const int row_bytes = d->cache.dim * (d->cache.dtype == THB_F32 ? 4 : 2), slots = 148 * (row_bytes <= 128 ? 4 : row_bytes <= 512 ? 2 : 1);
    const double base = (double)d->rows * d->cache.heads * c.head_tiles;
    const long span = d->window && d->window < d->max_len ? d->window + 15L : d->max_len;  // (from a multiple of 16 on)
    const long want = base >= slots ? 1 : (long)(slots / base);
    auto up = [](long v) { return v < 64 ? 64 : (v + 63) / 64 * 64; };
    long chunk = up((span + want - 1) / want);
    if (d->rows > 1 && chunk > 2048) chunk = 2048;
    long chunks = (span + chunk - 1) / chunk;
    // A cluster saves the second launch, but its CTAs come and go together: one wave of them, and of clusters of sixteen one to each
    // of the device's eight parts (two there took turns: 34 us instead of 23 for sixteen of them); and where it leaves a CTA no more than
    // 256 tokens, or no more than two launches would.
    c.cluster = 0;
    const int most = base <= 8 ? 16 : 8;
    long n = 2;
    while (n < most && base * n * 2 <= slots && n * 64 < span) n *= 2;
    const long clustered = up((span + n - 1) / n);
    if (chunks > 1 && base * n <= slots && clustered <= (chunk > 256 ? chunk : 256)) {
        chunks = n;
        chunk = clustered;
        c.cluster = 1;
    }
    c.chunk = (int)chunk;
    c.chunks = chunks < 1 ? 1 : (int)(chunks < (1L << 30) ? chunks : 1L << 30);
    return c;
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
    if (d->q_heads % d->cache.heads) return 0;
    const Cut c = cut_of(d);
    return c.chunks == 1 || c.cluster ? 0 : (size_t)d->rows * c.chunks * d->q_heads * (d->cache.dim + 2) * sizeof(float);
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
    const Cut c = cut_of(d);
    const AttnParams p = {d->cache, d->len, d->seq, q, y, d->lse, (float *)d->scratch, d->rows, d->q_heads, d->q_ld, d->y_ld, d->max_len, d->window,
                          d->q_heads / d->cache.heads, c.head_tiles, c.chunk, c.chunks, c.cluster, d->scale};
    if (p.rows > 65535 || p.chunks > 65535 || (long)p.rows * p.q_heads >= 1L << 31)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_paged_attn_fwd: more rows, chunks or heads than a launch has blocks");
    if (d->scratch_bytes < thb_paged_attn_scratch(d) || (p.chunks > 1 && !p.cluster && (!d->scratch || thb_misaligned(d->scratch))))
        return thb_refuse(THB_ERR_ARG, "thb_paged_attn_fwd: scratch is missing, misaligned or smaller than thb_paged_attn_scratch says");
    switch (dtype) {
    case THB_F32: return launch_attn<float>(p, c.ht, (cudaStream_t)s);
    case THB_F16: return launch_attn<__half>(p, c.ht, (cudaStream_t)s);
    default: return launch_attn<__nv_bfloat16>(p, c.ht, (cudaStream_t)s);
    }
}
