// 4-bit Linear on N <= 8 rows: y[n][m] = act(scale[m] * x_scale[n] * sum_k x[n][k] (q[m][k] - z[m][k/g]) s[m][k/g] + shift[m]).
// HBM-bound on the codes (half a byte a weight): at 6.5 TB/s 13 T weights arrive a second, 2.7 instructions of a lane for each, fewer
// than eight rows of fused multiply-adds take.  So the products run on the tensor cores whatever N is, by mma.sync m16n8k16 (tcgen05's
// smallest tile is 128 x 8 with operands in shared memory or TMEM: the codes would pass through either once more for nothing): 16 rows of
// weights are the A operand, the rows of x the 8 columns of B.  The order of k in a product is free, so a lane's operands are what it
// loads: vectors of codes in the order in which they are stored.
// A code becomes q - z in 16 bits exactly (an integer of 5 bits): or'ed into the mantissa of 1024 (fp16; bf16: 128), then z + 1024 is
// subtracted.  Products and their sums are exact or fp32, a group's sum takes its scale in fp32.  x in fp32 is three bf16 parts
// (8 + 8 + 8 bits), each multiplied; e4m3 codes are fp16 numbers.
// What bounds it: waiting, with four warps to a scheduler (sixteen of 128 registers).  9 (fp16) or 11 (bf16) instructions unpack 8 weights and as
// many again do everything else, 12 us of issue for the 4096->32003 below, but issue is busy in 32 to 53 % of the cycles only, the integer pipe in
// 25 to 49 %.  Where rows are few a warp has 2 to 7 blocks in all: the latency of its first stage (the second is not asked for until x is staged),
// of scales that are asked for two blocks ahead, and of the parts' exchange is most of the time; of the 4096->32003's 8.7 cycles an instruction 1.8 are
// the exchange's barriers and 1.6 global loads.  us a call in a chain (of the measured copy rate): 4096->128000, one row, bf16 groups of 128 55.2
// (4.9 TB/s, 75 %); 4096->32003, four rows of e4m3, groups of 32 with zero points 29.8 (40 %); 14336->4096, one row, fp16 11.1 (42 %); 9216->4096, eight rows,
// bf16 groups of 64 with zero points 10.8 (30 %); 25088->4096, three rows, fp32 33.6 (24 %: each row's values are three parts and three products,
// on five empty columns of eight).  Variants for fp32 rows beyond the shared memory and zero points spill 200 to 376 bytes of registers.
// Before: codes straight from global memory into registers 164 us for the 4096->32003, x in registers and tiles of 16 rows 31.  Tried and
// slower: an equal share of a CTA's blocks for each warp, across tiles (a block or two less a warp, but 0.2 to 4 us more a call for where parts
// begin and how they are joined); fp32 vectors taken apart by a warp's lanes together and handed on through shared memory (36 for 32).
#include "tokens.cuh"
#include <cuda_fp8.h>

namespace {

struct Q4Params {
    const void *x;
    const float *x_scale;
    const uint8_t *w, *wzero;
    const void *wscale;
    const float *scale, *shift;
    void *y;
    thb_act act;
    int N, K, M, x_ld, y_ld, w_ld, s_ld, z_ld, s_dtype, dtype;
};

struct XF16 { static constexpr bool BF = false; static constexpr int PARTS = 1, SIZE = 2; };
struct XBF16 { static constexpr bool BF = true; static constexpr int PARTS = 1, SIZE = 2; };
struct XF32 { static constexpr bool BF = true; static constexpr int PARTS = 3, SIZE = 4; };
struct XE4M3 { static constexpr bool BF = false; static constexpr int PARTS = 1, SIZE = 1; };

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// c = a b: a group's first product
template <bool BF>
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// 8 rows of 16 bytes four times: lane (g, t) gets word t of rows g, g + 8, g + 16 and g + 24, whose addresses lanes 0 to 31 give
__device__ __forceinline__ void codes_of(uint32_t (&w)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}

// (a & mask) | base in one instruction
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t mask, uint32_t base)
{
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(base));
    return d;
}
// the zero point of a row's group (byte i of four) as what is subtracted from a pair: z + 1024 (fp16) or z + 128 (bf16) twice
template <bool BF> __device__ __forceinline__ uint32_t zero_pair(uint32_t z, int i) { return __byte_perm(z, BF ? 0x43u : 0x64u, 0x4040 + i * 0x0101); }
// codes (0, 4), (1, 5), (2, 6), (3, 7) of a word (nibbles, lowest first) less the zero point, as pairs of 16-bit numbers.  In fp16 the odd
// ones are taken where they stand, as 1024 + 16 q, and scaled by the subtraction of 64 + z.
template <bool BF> __device__ __forceinline__ void pairs_of(uint32_t word, uint32_t za, uint32_t zb, uint32_t (&d)[4])
{
    if constexpr (BF) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t v = code_pair(word >> (4 * i), 0x000f000fu, 0x43004300u);
            const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&za));
            d[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t u = i ? word >> 8 : word, v = code_pair(u, 0x000f000fu, 0x64006400u), w = code_pair(u, 0x00f000f0u, 0x64006400u);
            const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&za));
            const __half2 k = __hfma2(*reinterpret_cast<const __half2 *>(&w), __float2half2_rn(0.0625f), *reinterpret_cast<const __half2 *>(&zb));
            d[i] = *reinterpret_cast<const uint32_t *>(&h);
            d[i + 1] = *reinterpret_cast<const uint32_t *>(&k);
        }
    }
}
// -(64 + z) from 1024 + z
__device__ __forceinline__ uint32_t zero_pair_16(uint32_t za)
{
    const __half2 d = __hsub2(__float2half2_rn(960.f), *reinterpret_cast<const __half2 *>(&za));
    return *reinterpret_cast<const uint32_t *>(&d);
}

// What a lane holds of 8 consecutive values of its row of x, as loaded and as four B registers a part: (x0,x4), (x1,x5), (x2,x6), (x3,x7)
template <typename X> struct XVec;
struct XVec16 {
    uint4 v;
    __device__ __forceinline__ void load(const uint8_t *x, int k, int K)
    {
        v = make_uint4(0, 0, 0, 0);
        if (k < K) v = *reinterpret_cast<const uint4 *>(x + 2L * k);
    }
    __device__ __forceinline__ void cut(int left)  // values from `left` on (0 < left < 8) lie behind the row
    {
        uint32_t *h = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] &= 2 * i + 1 < left ? 0xffffffffu : 2 * i < left ? 0xffffu : 0u;
    }
    __device__ __forceinline__ void get(uint32_t (&b)[1][4]) const
    {
        b[0][0] = __byte_perm(v.x, v.z, 0x5410);
        b[0][1] = __byte_perm(v.x, v.z, 0x7632);
        b[0][2] = __byte_perm(v.y, v.w, 0x5410);
        b[0][3] = __byte_perm(v.y, v.w, 0x7632);
    }
};
template <> struct XVec<XF16> : XVec16 {};
template <> struct XVec<XBF16> : XVec16 {};
template <> struct XVec<XE4M3> {
    uint2 v;
    static __device__ __forceinline__ uint32_t two(uint32_t codes)  // two codes in the low halfword -> two fp16
    {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
        return (uint32_t)h.x | (uint32_t)h.y << 16;
    }
    __device__ __forceinline__ void load(const uint8_t *x, int k, int K)
    {
        v = make_uint2(0, 0);
        if (k < K) v = *reinterpret_cast<const uint2 *>(x + k);
    }
    __device__ __forceinline__ void cut(int left)
    {
        v.x &= left >= 4 ? 0xffffffffu : (1u << 8 * left) - 1;
        v.y &= left <= 4 ? 0u : (1u << 8 * (left - 4)) - 1;
    }
    __device__ __forceinline__ void get(uint32_t (&b)[1][4]) const
    {
        const uint32_t p = __byte_perm(v.x, v.y, 0x5140), r = __byte_perm(v.x, v.y, 0x7362);  // codes 0 4 1 5 and 2 6 3 7
        b[0][0] = two(p);
        b[0][1] = two(p >> 16);
        b[0][2] = two(r);
        b[0][3] = two(r >> 16);
    }
};
template <> struct XVec<XF32> {
    float v[8];
    __device__ __forceinline__ void load(const uint8_t *x, int k, int K)
    {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k + 4 * h < K) f = *reinterpret_cast<const float4 *>(x + 4L * (k + 4 * h));
            v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
        }
    }
    __device__ __forceinline__ void cut(int left)
    {
#pragma unroll
        for (int i = 1; i < 8; i++) v[i] = i < left ? v[i] : 0.f;
    }
    // A part is the top 16 bits of what the parts before it leave: 8 bits of mantissa each, no rounding, the rest is exact.  (The rest of an
    // infinity is zero, not NaN: looked at where one of the eight times zero is not zero.)
    __device__ __forceinline__ void get(uint32_t (&b)[3][4]) const
    {
        uint32_t part[3][8];
        float zero = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) zero = fmaf(v[i], 0.f, zero);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            part[0][i] = __float_as_uint(v[i]);
#pragma unroll
            for (int q = 1; q < 3; q++)
                part[q][i] = __float_as_uint(__uint_as_float(part[q - 1][i]) - __uint_as_float(part[q - 1][i] & 0xffff0000u));
        }
        if (zero != 0.f)
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (isinf(v[i])) part[1][i] = part[2][i] = 0;
#pragma unroll
        for (int q = 0; q < 3; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) b[q][i] = __byte_perm(part[q][i], part[q][i + 4], 0x7632);
    }
};

// How a launch is cut, by the shape alone: the warps of a CTA are wk along k times WARPS / wk tiles of 32 rows, `mine` blocks of 128 k each.
struct Q4Cut {
    int wk, mine, tiles, wide;  // wide: 16-bit scales, and zero points, are aligned to what a block has of them (1), or to SG (2)
};
constexpr int WARPS = 16, NB = 2, STAGES = 2;     // blocks a stage; stages a warp
constexpr int STAGE = NB * 2048;                  // bytes: 32 rows
constexpr int COL = 36, PITCH = 8 * COL;          // floats a column, and a warp's part, take in shared memory: no bank twice in the parts' writes
constexpr int RING = WARPS * STAGES * STAGE, PARTS_AT = RING, SCALES_AT = PARTS_AT + WARPS * PITCH * 4;
constexpr int SG = 8, SP = 12;                    // groups a row whose scales a warp has at a time; words that they and their zero points take
constexpr int X_AT = SCALES_AT + WARPS * 32 * SP * 4, X_MOST = 227 * 1024 - 1024 - X_AT;  // x in operand order, where it fits

// One CTA of sixteen warps to an SM owns a range of tiles.  The codes come through a ring of a warp's own in shared memory, 32 rows by two
// blocks a stage, by cp.async of 16 bytes (no registers, no barrier between warps: 64 KB under way an SM while as much is multiplied).  x comes
// in operand order from shared memory, or where it does not fit from the L1, a block ahead, and each of its operands is multiplied by both
// 16-row halves of the tile.  Where the tiles are too few for the warps, wk of them share a row's blocks and their parts are added through shared memory; else a warp has whole rows.
// Lane (g = lane / 4, t = lane % 4) holds rows g, g + 8, g + 16 and g + 24.  Of each 32 k it takes the 8 of its t, word t of 16 bytes: what ldmatrix
// gives it of four times eight rows.
template <typename X, int GROUP, bool ZEROS, bool XS>
__global__ void __launch_bounds__(WARPS * 32, 1) gemv_q4_kernel(Q4Params p, Q4Cut cut)
{
    constexpr int VW = GROUP / 32, NG = 128 / GROUP, SB = SG / NG;  // words of a lane's row a group, groups a block, blocks whose scales are at hand
    // A block's codes are read at once where x comes from the L1 (11008->11000 on four rows 27.5 -> 25.0 us) or a group is a block (4096->128000
    // 54.5 -> 53.9); else as they are needed, for the registers' sake (4096->32003 in e4m3, groups of 32, 28.8 -> 28.3).
    constexpr bool AHEAD = !XS || NG == 1;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * STAGES * STAGE;
    const int tile0 = (int)((long)cut.tiles * blockIdx.x / gridDim.x), tile1 = (int)((long)cut.tiles * (blockIdx.x + 1) / gridDim.x);
    const int wk = cut.wk, wm = WARPS / wk, kw = warp % wk, mw = warp / wk;
    const int blocks = (p.K + 127) / 128, groups = (p.K + GROUP - 1) / GROUP, bytes = ((p.K + 1) / 2 + 15) / 16 * 16;
    const int b0 = kw * cut.mine, b1 = min(blocks, b0 + cut.mine);  // (b0 may be beyond the row: then there is nothing to add)

    // 16-byte pieces of a stage, permuted so that no load of 8 rows meets a bank twice
    auto piece = [](int row, int c) { return ((row * 8 + c) ^ (row & 7)) * 16; };

    // ---- the codes' loads, a stage ahead of the products; lane: pieces fc of rows fr, fr + 4, ...
    const int fr = lane >> 3, fc = lane & 7;
    int ftile = tile0 + mw, fb = b0, fslot = 0;
    const uint8_t *fsrc = p.w;
    long frow = 0;
    const uint32_t fto = ring + piece(fr, fc), fto4 = ring + piece(fr + 4, fc) - 512;  // (rows i * 4 + fr: even and odd i)
    auto seek = [&] {
        const bool any = ftile < tile1 && fb + (fc >> 2) < b1;
        fsrc = any ? p.w + (long)(ftile * 32 + fr) * p.w_ld + fb * 64 + fc * 16 : p.w;
        frow = any ? 4L * p.w_ld : 0;
    };
    seek();
    auto fetch = [&] {
        const int o = fb * 64 + fc * 16;
        const uint32_t size = ftile < tile1 && fb + (fc >> 2) < b1 && o < bytes ? 16 : 0, at = fslot * STAGE;
        const uint8_t *src = size ? fsrc : p.w;
        if (ftile * 32 + 32 <= p.M) {
            const long step = size ? frow : 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                cp_async16((i & 1 ? fto4 : fto) + at + i * 512, src, size);
                src += step;
            }
        } else {  // (rows beyond the last are zeros and not written)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool row = size && ftile * 32 + i * 4 + fr < p.M;
                cp_async16((i & 1 ? fto4 : fto) + at + i * 512, row ? src + i * frow : p.w, row ? 16 : 0);
            }
        }
        cp_async_commit();
        fslot ^= 1;
        fb += NB;
        fsrc += NB * 64;
        if (fb >= b1) {
            fb = b0;
            ftile += wm;
            seek();
        }
    };
    // ---- the scales and zero points of SG groups (SB blocks): a lane loads those of row `lane`, SB blocks ahead and as they lie in memory (16
    // bits: two to a word where they are aligned), and puts them into the warp's shared memory as floats and as bytes
    float *const scales = reinterpret_cast<float *>(smem + SCALES_AT) + warp * 32 * SP;
    uint32_t sn[SG], zn[SG];
#pragma unroll
    for (int i = 0; i < SG; i++) sn[i] = zn[i] = 0;
    auto fetch_scales = [&](int tile, int b) {
        const int group = b * NG, left = min(groups, b1 * NG) - group;
        const long row = tile * 32 + lane;
        if (tile >= tile1 || row >= p.M || left <= 0) return;
        const long at = row * p.s_ld + group;
        const uint8_t *z = ZEROS ? p.wzero + row * p.z_ld + group : nullptr;
        if (cut.wide == 2 && left >= SG) {
            const uint4 v = *reinterpret_cast<const uint4 *>((const uint16_t *)p.wscale + at);
            sn[0] = v.x; sn[1] = v.y; sn[2] = v.z; sn[3] = v.w;
            if (ZEROS) {
                const uint2 u = *reinterpret_cast<const uint2 *>(z);
                zn[0] = u.x; zn[1] = u.y;
            }
        } else if (cut.wide && NG > 1) {
#pragma unroll
            for (int n = 0; n < SB; n++) {
                if (n * NG >= left) break;
                const uint16_t *s = (const uint16_t *)p.wscale + at + n * NG;
                if constexpr (NG == 4) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(s);
                    sn[2 * n] = v.x; sn[2 * n + 1] = v.y;
                    if (ZEROS) zn[n] = *reinterpret_cast<const uint32_t *>(z + n * NG);
                } else {
                    sn[n] = *reinterpret_cast<const uint32_t *>(s);
                    if (ZEROS) zn[n] = *reinterpret_cast<const uint16_t *>(z + n * NG);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < SG; i++)
                if (i < left) {
                    sn[i] = p.s_dtype == THB_F32 ? ((const uint32_t *)p.wscale)[at + i] : ((const uint16_t *)p.wscale)[at + i];
                    if (ZEROS) zn[i] = z[i];
                }
        }
    };
    auto put_scales = [&](int b) {
        const int left = min(groups, b1 * NG) - b * NG;
        const bool full = cut.wide == 2 && left >= SG, packed = full || (cut.wide && NG > 1);
        float f[SG];
        if (p.s_dtype == THB_F32) {
#pragma unroll
            for (int i = 0; i < SG; i++) f[i] = __uint_as_float(sn[i]);
        } else {
            uint32_t h[SG];
#pragma unroll
            for (int i = 0; i < SG; i++) h[i] = packed ? sn[i / 2] >> (16 * (i & 1)) : sn[i];
            if (p.s_dtype == THB_F16) {
#pragma unroll
                for (int i = 0; i < SG; i++) f[i] = __half2float(__ushort_as_half((unsigned short)h[i]));
            } else {
#pragma unroll
                for (int i = 0; i < SG; i++) f[i] = __uint_as_float(h[i] << 16);
            }
        }
        if (left < SG)  // (what lies behind a row's groups is not a scale; rows behind the last have any, and are not written)
#pragma unroll
            for (int i = 0; i < SG; i++)
                if (i >= left) f[i] = 0.f;
        float *to = scales + lane * SP;
        *reinterpret_cast<float4 *>(to) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4 *>(to + 4) = make_float4(f[4], f[5], f[6], f[7]);
        if (ZEROS) {
            uint2 z = make_uint2(zn[0], zn[1]);
            if (!full && packed && NG == 2) z = make_uint2((zn[0] & 0xffffu) | zn[1] << 16, (zn[2] & 0xffffu) | zn[3] << 16);
            if (!packed) z = make_uint2(zn[0] | zn[1] << 8 | zn[2] << 16 | zn[3] << 24, zn[4] | zn[5] << 8 | zn[6] << 16 | zn[7] << 24);
            *reinterpret_cast<uint2 *>(to + SG) = make_uint2(z.x & 0x0f0f0f0fu, z.y & 0x0f0f0f0fu);
        }
    };

    // ---- x: in operand order in shared memory, put there once a CTA, or where it does not fit the four vectors of a lane from the L1, each
    // loaded again for the next block as soon as it has been taken
    const uint8_t *const xrow = (const uint8_t *)p.x + (long)(g < p.N ? g : 0) * p.x_ld * X::SIZE;
    const int xk = g < p.N ? p.K : 0;  // (columns beyond the rows of x are zeros)
    XVec<X> xv[4];
    auto x_at = [&](int b, int i, int tt) { return b * 128 + i * 32 + tt * 8; };
    uint4 *const xs = reinterpret_cast<uint4 *>(smem + X_AT);  // [block][vector][part][N][t], then a zero for the lanes beyond the rows
    const int xstep = g < p.N ? p.N * 4 : 0;
    const uint4 *const xmine = g < p.N ? xs + g * 4 + t : xs + blocks * 4 * X::PARTS * p.N * 4;

    // Codes, scales and zero points may be what the launch before has written, which only the wait in pdl_enter() makes visible: nothing of them
    // is read ahead of it, and none through the non-coherent path, whose data has to stay as it is for as long as a kernel runs.
    pdl_enter();
    fetch();
    fetch_scales(tile0 + mw, b0);
    if constexpr (XS) {
        for (int e = tid; e < blocks * 16 * p.N; e += WARPS * 32) {
            const int tt = e & 3, n = (e >> 2) % p.N, i = (e >> 2) / p.N & 3, b = (e >> 2) / p.N >> 2, k = x_at(b, i, tt);
            XVec<X> v;
            v.load((const uint8_t *)p.x + (long)n * p.x_ld * X::SIZE, k, p.K);
            if (p.K - k > 0 && p.K - k < 8) v.cut(p.K - k);
            uint32_t r[X::PARTS][4];
            v.get(r);
#pragma unroll
            for (int q = 0; q < X::PARTS; q++) xs[(((b * 4 + i) * X::PARTS + q) * p.N + n) * 4 + tt] = make_uint4(r[q][0], r[q][1], r[q][2], r[q][3]);
        }
        if (tid == 0) xs[blocks * 4 * X::PARTS * p.N * 4] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) xv[i].load(xrow, x_at(b0, i, t), xk);
    }

    // where row `lane` lies in a stage: pieces differ in bits 4 to 6 by what their number differs in
    const uint32_t lane_at = ring + piece(lane, 0);
    int slot = 0;
    for (int step = tile0; step < tile1; step += wm) {
        const int tile = step + mw;
        float acc[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) acc[i][q] = 0.f;
        if (tile < tile1 && b0 < b1)
            for (int b = b0; b < b1; b += NB) {
                __syncwarp();  // (all lanes have read the last stage and its scales)
                if ((b - b0) % SB == 0) {
                    put_scales(b);
                    const bool wraps = b + SB >= b1;
                    fetch_scales(wraps ? tile + wm : tile, wraps ? b0 : b + SB);
                }
                fetch();
                cp_async_wait<STAGES - 1>();
                __syncwarp();
                const uint32_t at = lane_at + slot * STAGE;
                slot ^= 1;
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    if (b + n >= b1) break;
                    const int next = b + n + 1 < b1 ? b + n + 1 : b0, sb = (b - b0) % SB + n;
                    const uint4 *const xblock = xmine + (b + n) * 4 * X::PARTS * xstep;
                    if (!XS && (b + n) * 128 + 128 > p.K)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int left = p.K - x_at(b + n, i, t);
                            if (left > 0 && left < 8) xv[i].cut(left);
                        }
                    uint32_t w[4][4];
                    if (AHEAD)
#pragma unroll
                        for (int i = 0; i < 4; i++) codes_of(w[i], at ^ (n * 4 + i) * 16);
                    // the block's scales and zero points of the lane's four rows
                    float sc[4][NG];
                    uint32_t zs[4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float *from = scales + (g + 8 * r) * SP;
                        if constexpr (NG == 4) {
                            const float4 v = *reinterpret_cast<const float4 *>(from + sb * NG);
                            sc[r][0] = v.x; sc[r][1 % NG] = v.y; sc[r][2 % NG] = v.z; sc[r][3 % NG] = v.w;
                        } else
#pragma unroll
                            for (int j = 0; j < NG; j++) sc[r][j] = from[sb * NG + j];
                        if (ZEROS) zs[r] = reinterpret_cast<const uint32_t *>(from)[SG + sb * NG / 4];
                    }
#pragma unroll
                    for (int j = 0; j < NG; j++) {
                        float c[2][4];
                        uint32_t za[4], zb[4];
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            za[r] = ZEROS ? zero_pair<X::BF>(zs[r], sb * NG % 4 + j) : X::BF ? 0x43084308u : 0x64086408u;
                            zb[r] = X::BF ? 0 : zero_pair_16(za[r]);
                        }
#pragma unroll
                        for (int h = 0; h < VW; h++) {
                            uint32_t xb[X::PARTS][4];
                            if (!AHEAD) codes_of(w[j * VW + h], at ^ (n * 4 + j * VW + h) * 16);
                            if constexpr (XS) {
#pragma unroll
                                for (int q = 0; q < X::PARTS; q++) {
                                    const uint4 v = xblock[((j * VW + h) * X::PARTS + q) * xstep];
                                    xb[q][0] = v.x; xb[q][1] = v.y; xb[q][2] = v.z; xb[q][3] = v.w;
                                }
                            } else {
                                xv[j * VW + h].get(xb);
                                xv[j * VW + h].load(xrow, x_at(next, j * VW + h, t), xk);
                            }
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                uint32_t a[2][4];
#pragma unroll
                                for (int r = 0; r < 2; r++) pairs_of<X::BF>(w[j * VW + h][2 * i + r], za[2 * i + r], zb[2 * i + r], a[r]);
#pragma unroll
                                for (int q = X::PARTS - 1; q >= 0; q--) {
                                    if (h == 0 && q == X::PARTS - 1) mma16816_first<X::BF>(c[i], a[0][0], a[1][0], a[0][1], a[1][1], xb[q][0], xb[q][1]);
                                    else mma16816<X::BF>(c[i], a[0][0], a[1][0], a[0][1], a[1][1], xb[q][0], xb[q][1]);
                                    mma16816<X::BF>(c[i], a[0][2], a[1][2], a[0][3], a[1][3], xb[q][2], xb[q][3]);
                                }
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 2; i++)
#pragma unroll
                            for (int q = 0; q < 4; q++) acc[i][q] = fmaf(c[i][q], sc[2 * i + (q >> 1)][j], acc[i][q]);
                    }
                }
            }
        // the results.  acc[i]: rows 16i + g (twice) and 16i + g + 8, columns 2t and 2t + 1
        auto finish = [&](int n, int m, float v) {
            if (n >= p.N || m >= (p.M + 7) / 8 * 8 || (p.dtype == THB_F32 && m >= (p.M + 3) / 4 * 4)) return;
            if (m < p.M) {
                if (p.x_scale) v *= p.x_scale[n];
                if (p.scale) v *= p.scale[m];
                if (p.shift) v += p.shift[m];
                if (p.act.kind != THB_ACT_NONE)
                    v = thb_apply_act(v, p.act.kind, p.act.threshold, p.act.value, p.act.alpha, p.act.kind == THB_ACT_PRELU ? p.act.slope[m] : 0.f);
            } else
                v = 0.f;  // channels of the padded tail of y are kept at exact zero
            const long to = (long)n * p.y_ld + m;
            if (p.dtype == THB_F32) ((float *)p.y)[to] = v;
            else if (p.dtype == THB_F16) ((__half *)p.y)[to] = __float2half_rn(v);
            else ((__nv_bfloat16 *)p.y)[to] = __float2bfloat16_rn(v);
        };
        // A warp's sums go through its part of shared memory, so that the four of a lane's columns become rows side by side.
        float *const parts = reinterpret_cast<float *>(smem + PARTS_AT);
        float *mypart = parts + warp * PITCH;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) mypart[(2 * t + (q & 1)) * COL + i * 16 + g + (q >> 1) * 8] = acc[i][q];
        if (wk == 1) {
            __syncwarp();
            if (tile < tile1)
                for (int n = 0; n < p.N; n++) finish(n, tile * 32 + lane, mypart[n * COL + lane]);
            __syncwarp();
        } else {
            __syncthreads();
            // a warp adds a column of a tile
            for (int i = warp; i < wm * 8; i += WARPS) {
                const int n = i % 8;
                if (n >= p.N || step + i / 8 >= tile1) continue;
                const float *from = parts + i / 8 * wk * PITCH + n * COL + lane;
                float v = 0.f;
                for (int q = 0; q < wk; q++) v += from[q * PITCH];
                finish(n, (step + i / 8) * 32 + lane, v);
            }
            __syncthreads();
        }
    }
    cp_async_wait<0>();
}

template <typename X, int GROUP, bool ZEROS, bool XS> int launch_q4_kernel(const Q4Params &p, const Q4Cut &c, int grid, int dev, cudaStream_t st)
{
    const auto kern = gemv_q4_kernel<X, GROUP, ZEROS, XS>;
    static bool set[64];
    if (!set[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, XS ? X_AT + X_MOST : X_AT);
        if (e != cudaSuccess) return thb_note_launch(e, "gemv_q4_kernel attributes");
        set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = X_AT + (XS ? (p.K + 127) / 128 * 256 * X::PARTS * p.N + 16 : 0);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = thb_pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, c);
    return thb_note_launch(e != cudaSuccess ? e : cudaGetLastError(), "gemv_q4_kernel");
}

template <typename X, int GROUP, bool ZEROS> int launch_q4_group(const Q4Params &p, cudaStream_t st)
{
    constexpr int NG = 128 / GROUP;
    const int sms = thb_sm_count();
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: device ordinal above 63");
    Q4Cut c;
    const int blocks = (p.K + 127) / 128;
    c.tiles = (p.M + 31) / 32;
    // As few warps to a row as keep a CTA's warps equally busy: the blocks that a warp takes one after the other, and two more a tile for the
    // parts' exchange.
    const int grid = c.tiles < sms ? c.tiles : sms, most = (c.tiles + grid - 1) / grid;
    long best = 0;
    for (int wk = 1; wk <= WARPS && (wk == 1 || wk < 2 * blocks); wk *= 2) {
        const long steps = (most + WARPS / wk - 1) / (WARPS / wk), cost = steps * ((blocks + wk - 1) / wk + (wk > 1 ? 2 : 0));
        if (wk == 1 || cost < best) {
            best = cost;
            c.wk = wk;
        }
    }
    c.mine = (blocks + c.wk - 1) / c.wk;
    auto aligned = [&](int n) {
        return p.s_dtype != THB_F32 && p.s_ld % n == 0 && reinterpret_cast<uintptr_t>(p.wscale) % (2 * n) == 0 &&
               (!p.wzero || (p.z_ld % n == 0 && reinterpret_cast<uintptr_t>(p.wzero) % n == 0));
    };
    // (a warp's first block is a multiple of mine)
    c.wide = aligned(SG) && (c.wk == 1 || c.mine * NG % SG == 0) ? 2 : aligned(NG) ? 1 : 0;
    return (long)blocks * 256 * X::PARTS * p.N + 16 <= X_MOST ? launch_q4_kernel<X, GROUP, ZEROS, true>(p, c, grid, dev, st)
                                                              : launch_q4_kernel<X, GROUP, ZEROS, false>(p, c, grid, dev, st);
}

template <typename X> int launch_q4(const Q4Params &p, int group, cudaStream_t st)
{
    if (group == 32) return p.wzero ? launch_q4_group<X, 32, true>(p, st) : launch_q4_group<X, 32, false>(p, st);
    if (group == 64) return p.wzero ? launch_q4_group<X, 64, true>(p, st) : launch_q4_group<X, 64, false>(p, st);
    return p.wzero ? launch_q4_group<X, 128, true>(p, st) : launch_q4_group<X, 128, false>(p, st);
}

}  // namespace

extern "C" int thb_gemv_q4_fwd(const thb_gemv_q4_desc *d, const void *x, const float *x_scale, void *y, thb_stream s)
{
    if (!d) return THB_ERR_ARG;
    if (d->dtype != THB_F32 && d->dtype != THB_F16 && d->dtype != THB_BF16)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: dtype is not THB_F32, THB_F16 or THB_BF16");
    if (d->N < 0 || d->K < 1 || d->M < 1) return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: N < 0, K < 1 or M < 1");
    if (d->N > 8) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: more than 8 rows of x");
    if (d->group != 32 && d->group != 64 && d->group != 128)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: group is not 32, 64 or 128");
    if (d->wscale_dtype != THB_F32 && d->wscale_dtype != THB_F16 && d->wscale_dtype != THB_BF16)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: wscale_dtype is not THB_F32, THB_F16 or THB_BF16");
    if (d->K > (1 << 30) || d->M > (1 << 30)) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: K or M above 2^30");
    if (d->N == 0) return THB_OK;
    if (!x || !y || !d->w || !d->wscale) return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: x, y, w and wscale must be set");
    const int al = thb_channel_align(d->dtype), xal = x_scale ? 16 : al, groups = (d->K + d->group - 1) / d->group;
    if (thb_misaligned(x) || thb_misaligned(y) || thb_misaligned(d->w))
        return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: x, y or w is not 16-byte aligned");
    if (x == y) return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: y in the place of x");
    if (d->x_ld % xal || d->x_ld < d->K || d->y_ld % al || d->y_ld < d->M)
        return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: x_ld or y_ld is below the row or no multiple of the alignment");
    if (d->w_ld % 16 || d->w_ld < (d->K + 1) / 2 || d->s_ld < groups || (d->wzero && d->z_ld < groups))
        return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: w_ld is below the row or no multiple of 16, or s_ld or z_ld is below the groups of a row");
    if ((reinterpret_cast<uintptr_t>(d->wscale) & (d->wscale_dtype == THB_F32 ? 3 : 1)))
        return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: wscale is not aligned to its type");
    if (d->act.kind < THB_ACT_NONE || d->act.kind > THB_ACT_TANH || (d->act.kind == THB_ACT_PRELU && !d->act.slope))
        return thb_refuse(THB_ERR_ARG, "thb_gemv_q4_fwd: unknown activation, or THB_ACT_PRELU without slopes");
    const Q4Params p = {x, x_scale, d->w, d->wzero, d->wscale, d->scale, d->shift, y, d->act, d->N, d->K, d->M, d->x_ld, d->y_ld,
                        d->w_ld, d->s_ld, d->z_ld, d->wscale_dtype, d->dtype};
    if (x_scale) return launch_q4<XE4M3>(p, d->group, (cudaStream_t)s);
    switch (d->dtype) {
    case THB_F32: return launch_q4<XF32>(p, d->group, (cudaStream_t)s);
    case THB_F16: return launch_q4<XF16>(p, d->group, (cudaStream_t)s);
    default: return launch_q4<XBF16>(p, d->group, (cudaStream_t)s);
    }
}

extern "C" int thb_q4_quantize_host(const float *w, long M, int K, long ld, int group, int with_zero, unsigned char *codes, int w_ld, float *wscale,
                                    int s_ld, unsigned char *wzero, int z_ld)
{
    if (!w || !codes || !wscale || M < 1 || K < 1 || ld < K || group < 1 || w_ld < (K + 1) / 2 || (with_zero && !wzero)) return THB_ERR_ARG;
    const int groups = (K + group - 1) / group;
    if (s_ld < groups || (with_zero && z_ld < groups)) return THB_ERR_ARG;
    for (long m = 0; m < M; m++) {
        const float *row = w + m * ld;
        unsigned char *out = codes + m * (long)w_ld;
        for (int i = 0; i < w_ld; i++) out[i] = 0;
        for (int j = 0; j < groups; j++) {
            const int k0 = j * group, k1 = k0 + group < K ? k0 + group : K;
            float lo = 0.f, hi = 0.f;
            for (int k = k0; k < k1; k++) {
                if (!(row[k] - row[k] == 0.f)) return THB_ERR_ARG;  // (not finite)
                lo = row[k] < lo ? row[k] : lo;
                hi = row[k] > hi ? row[k] : hi;
            }
            // symmetric: codes 1..15 around 8; otherwise 0 is a code and [lo, hi] the fifteen steps around it
            float step;
            int zero = 8;
            if (with_zero) {
                step = (float)(((double)hi - lo) / 15);
                zero = step > 0.f ? (int)(-(double)lo / step + 0.5) : 8;
                zero = zero > 15 ? 15 : zero;
                wzero[m * (long)z_ld + j] = (unsigned char)zero;
            } else
                step = (hi > -lo ? hi : -lo) / 7;
            wscale[m * (long)s_ld + j] = step;
            for (int k = k0; k < k1; k++) {
                const double q = step > 0.f ? (double)row[k] / step : 0.0;
                int c = zero + (int)(q < 0 ? q - 0.5 : q + 0.5);
                c = c < 0 ? 0 : c > 15 ? 15 : c;
                out[k / 2] |= (unsigned char)(c << 4 * (k & 1));
            }
        }
    }
    return THB_OK;
}
