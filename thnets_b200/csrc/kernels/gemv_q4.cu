// 4-bit Linear on N <= 8 rows: y[n][m] = act(scale[m] * x_scale[n] * sum_k x[n][k] (q[m][k] - z[m][k/g]) s[m][k/g] + shift[m]).
// HBM-bound on the codes (half a byte a weight): at 6.5 TB/s 13 T weights arrive a second, 2.7 instructions of a lane for each, fewer
// than eight rows of fused multiply-adds take.  So the products run on the tensor cores whatever N is, by mma.sync m16n8k16 (tcgen05's
// smallest tile is 128 x 8 with operands in shared memory or TMEM: the codes would pass through either once more for nothing): 16 rows of
// weights are the A operand, the rows of x the 8 columns of B.  The order of k in a product is free, so a lane's operands are what it
// loads: vectors of codes in the order in which they are stored.
// A code becomes q - z in 16 bits exactly (an integer of 5 bits): or'ed into the mantissa of 1024 (fp16; bf16: 128), then z + 1024 is
// subtracted.  Products and their sums are exact or fp32, a group's sum takes its scale in fp32.  x in fp32 is three bf16 parts
// (8 + 8 + 8 bits), each multiplied; e4m3 codes are fp16 numbers.
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

struct XF16 { static constexpr bool BF = false; static constexpr int PARTS = 1; };
struct XBF16 { static constexpr bool BF = true; static constexpr int PARTS = 1; };
struct XF32 { static constexpr bool BF = true; static constexpr int PARTS = 3; };
struct XE4M3 { static constexpr bool BF = false; static constexpr int PARTS = 1; };

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

// (a & mask) | base in one instruction
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t mask, uint32_t base)
{
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(mask), "r"(base));
    return d;
}
// the zero point of a row's group as what is subtracted from a pair: z + 1024 (fp16) or z + 128 (bf16) twice
template <bool BF> __device__ __forceinline__ uint32_t zero_pair(uint32_t z) { return ((z & 15) | (BF ? 0x4300u : 0x6400u)) * 0x10001u; }
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
    __device__ __forceinline__ void load(const void *x, long row, int k, int K)
    {
        v = make_uint4(0, 0, 0, 0);
        if (k < K) v = *reinterpret_cast<const uint4 *>((const uint16_t *)x + row + k);
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
    __device__ __forceinline__ void load(const void *x, long row, int k, int K)
    {
        v = make_uint2(0, 0);
        if (k < K) v = *reinterpret_cast<const uint2 *>((const uint8_t *)x + row + k);
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
    __device__ __forceinline__ void load(const void *x, long row, int k, int K)
    {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k + 4 * h < K) f = *reinterpret_cast<const float4 *>((const float *)x + row + k + 4 * h);
            v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
        }
    }
    __device__ __forceinline__ void cut(int left)
    {
#pragma unroll
        for (int i = 1; i < 8; i++) v[i] = i < left ? v[i] : 0.f;
    }
    // A part is the top 16 bits of what the parts before it leave: 8 bits of mantissa each, no rounding, the rest is exact (that of an
    // infinity is zero, not NaN).
    __device__ __forceinline__ void get(uint32_t (&b)[3][4]) const
    {
        uint32_t part[3][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            part[0][i] = __float_as_uint(v[i]);
#pragma unroll
            for (int q = 1; q < 3; q++) {
                const float x = __uint_as_float(part[q - 1][i]), top = __uint_as_float(part[q - 1][i] & 0xffff0000u);
                part[q][i] = __float_as_uint(x == top ? 0.f : x - top);
            }
        }
#pragma unroll
        for (int q = 0; q < 3; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) b[q][i] = __byte_perm(part[q][i], part[q][i + 4], 0x7632);
    }
};

// How a launch is cut, by the shape alone: the warps of a CTA are wk along k times WARPS / wk tiles of 16 rows; a row's blocks of 128 k are
// walked in `chunks` passes of wk warps by `mine` blocks each.
struct Q4Cut {
    int wk, mine, chunks, tiles, wide;  // wide: 16-bit scales, and zero points, are aligned to what a lane loads of them
};
#ifndef Q4W
#define Q4W 8
#endif
static_assert(Q4W == 8, "two groups of four warps");
constexpr int WARPS = Q4W, Q4_ACC = 64;  // warps a CTA; tiles whose sums a CTA keeps between chunks
constexpr int COL = 20, PITCH = 8 * COL;  // floats a column, and a warp's part, take in shared memory: no bank twice in the parts' writes

template <typename X> struct Q4Shape {
    static constexpr int NB = (X::PARTS == 3 ? 16 : 32) / WARPS;  // blocks a stage at most
    static constexpr int STAGES = X::PARTS == 3 ? 8 : 4;
    static constexpr int SCALES = 2 * 16 * (NB * 4 + 4) * 4;      // bytes of scales and zero points a warp
    static constexpr int RING = WARPS * STAGES * NB * 1024, FIXED = RING + 2 * WARPS * PITCH * 4 + WARPS * SCALES;
};

// One CTA to an SM owns a range of tiles.  A warp keeps its part of x in registers as B operands and walks the CTA's
// tiles past it; the codes come through a ring of its own in shared memory, 16 rows by `mine` blocks a stage, by cp.async of 16 bytes (no
// registers and no barrier between warps: up to 128 KB under way an SM).  The warps' parts are added at a tile's end; where a row has
// more chunks than one, the sums stay in shared memory until the last, and x of the next chunk is loaded during the last tile of this one.
// Lane (g = lane / 4, t = lane % 4) holds rows g and g + 8.  Of a block it takes the k of its t: 32 in one vector where a group is 128
// long, 16 of each of two groups, 8 of each of four, so that a product's k are all of one group.
template <typename X, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(WARPS * 32, 1) gemv_q4_kernel(Q4Params p, Q4Cut cut)
{
    constexpr int NB = Q4Shape<X>::NB, STAGES = Q4Shape<X>::STAGES;
    constexpr int VW = GROUP / 32, NG = 128 / GROUP;             // words a load, groups a block
    constexpr int RS = 32 / (NB * 4);                            // rows a warp's cp.async covers (NB = 1: 8, 2: 4, 4: 2)
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    float *part = reinterpret_cast<float *>(smem + Q4Shape<X>::RING);  // [2][warps][PITCH]
    float *sums = reinterpret_cast<float *>(smem + Q4Shape<X>::FIXED);  // [tiles of the CTA][128], where there are chunks
    const uint32_t ring = smem_u32(smem) + warp * STAGES * NB * 1024;

    const int tile0 = (int)((long)cut.tiles * blockIdx.x / gridDim.x), tile1 = (int)((long)cut.tiles * (blockIdx.x + 1) / gridDim.x);
    const int wk = cut.wk, wm = WARPS / wk, kw = warp % wk, mw = warp / wk;
    const int steps = (tile1 - tile0 + wm - 1) / wm;
    const int groups = (p.K + GROUP - 1) / GROUP, bytes = ((p.K + 1) / 2 + 15) / 16 * 16;

    // 16-byte pieces of a stage, permuted so that no load of 8, 4 or 2 rows meets a bank twice (rows of 64 bytes lie two to a line)
    auto piece = [](int row, int c) {
        const int at = row * (NB * 4) + c, line = at >> 3;
        const int f = VW == 4 ? (NB >= 2 ? (row & 1) << 2 : 0) : VW == 2 ? (NB >= 2 ? (row & 3) << 1 : (line & 1) << 1) : (NB >= 2 ? row & 7 : line & 3);
        return (at ^ f) * 16;
    };

    // ---- the codes' loads, STAGES - 1 units (a tile of a chunk) ahead
    int ftile = tile0 + mw, fchunk = 0, fslot = 0;
    const int fr = lane / (NB * 4), fc = lane % (NB * 4);
    const uint8_t *fsrc = p.w;
    long fstep = 0, fnext = 0;
    uint32_t fsize = 0;
    auto seek = [&] {
        const int o = (fchunk * wk + kw) * cut.mine * 64 + fc * 16;
        const bool in = fchunk < cut.chunks && fc < cut.mine * 4 && o < bytes;
        fsize = in ? 16 : 0;
        fsrc = in ? p.w + (long)(ftile * 16 + fr) * p.w_ld + o : p.w;
        fstep = in ? (long)RS * p.w_ld : 0;
        fnext = in ? (long)(wm - 1) * 16 * p.w_ld : 0;
    };
    seek();
    auto fetch = [&] {
        const uint32_t at = ring + fslot * (NB * 1024);
        if (ftile < tile1 && ftile * 16 + 16 <= p.M) {
#pragma unroll
            for (int i = 0; i < 16 / RS; i++) {
                cp_async16(at + piece(i * RS + fr, fc), fsrc, fsize);
                fsrc += fstep;
            }
        } else {  // (rows beyond the last are zeros and not written)
#pragma unroll
            for (int i = 0; i < 16 / RS; i++) {
                const bool in = ftile < tile1 && ftile * 16 + i * RS + fr < p.M;
                cp_async16(at + piece(i * RS + fr, fc), in ? fsrc : p.w, in ? fsize : 0);
                fsrc += fstep;
            }
        }
        fsrc += fnext;
        cp_async_commit();
        fslot = fslot + 1 == STAGES ? 0 : fslot + 1;
        ftile += wm;
        if (ftile - mw >= tile0 + steps * wm) {
            ftile = tile0 + mw;
            fchunk++;
            seek();
        }
    };
    // ---- the scales and zero points of a unit: lane l loads GL of row l / 2 one unit ahead, as they lie in memory (16 bits: two to a word
    // where they are aligned), and puts them into the warp's shared memory as floats and as pairs to subtract
    constexpr int GU = NB * NG, GL = GU / 2 > 0 ? GU / 2 : 1, SP = GU + 4;  // groups a unit, a lane; words a row
    float *const scales = reinterpret_cast<float *>(smem + Q4Shape<X>::FIXED - WARPS * Q4Shape<X>::SCALES) + warp * (Q4Shape<X>::SCALES / 4);
    uint32_t *const zeros = reinterpret_cast<uint32_t *>(scales) + 16 * SP;
    uint32_t sn[GL], zn[GL];
#pragma unroll
    for (int i = 0; i < GL; i++) sn[i] = zn[i] = 0;
    const int sj = GU > 1 ? (lane & 1) * GL : 0;
    auto fetch_scales = [&](int chunk, int tile) {
        const int group = (chunk * wk + kw) * cut.mine * NG + sj;
        const long row = tile * 16 + (lane >> 1);
        if (chunk >= cut.chunks || tile >= tile1 || row >= p.M || group >= groups) return;
        const long at = row * p.s_ld + group;
        if (cut.wide) {
            const uint16_t *s = (const uint16_t *)p.wscale + at;
            if constexpr (GL == 8) {
                const uint4 v = __ldg(reinterpret_cast<const uint4 *>(s));
                sn[0] = v.x; sn[1 % GL] = v.y; sn[2 % GL] = v.z; sn[3 % GL] = v.w;
            } else if constexpr (GL == 4) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(s));
                sn[0] = v.x; sn[1 % GL] = v.y;
            } else if constexpr (GL == 2)
                sn[0] = __ldg(reinterpret_cast<const uint32_t *>(s));
            else
                sn[0] = __ldg(s);
        } else {
#pragma unroll
            for (int i = 0; i < GL; i++)
                if (group + i < groups) sn[i] = p.s_dtype == THB_F32 ? __ldg((const uint32_t *)p.wscale + at + i) : __ldg((const uint16_t *)p.wscale + at + i);
        }
        if (ZEROS) {
            const uint8_t *z = p.wzero + row * p.z_ld + group;
            if (cut.wide && GL == 8) {
                const uint2 v = __ldg(reinterpret_cast<const uint2 *>(z));
                zn[0] = v.x; zn[1 % GL] = v.y;
            } else if (cut.wide && GL == 4)
                zn[0] = __ldg(reinterpret_cast<const uint32_t *>(z));
            else if (cut.wide && GL == 2)
                zn[0] = __ldg(reinterpret_cast<const uint16_t *>(z));
            else {
#pragma unroll
                for (int i = 0; i < GL; i++)
                    if (group + i < groups) zn[i] = __ldg(z + i);
            }
        }
    };
    auto put_scales = [&](int chunk) {
        const int group = (chunk * wk + kw) * cut.mine * NG + sj;
        float f[GL];
        if (p.s_dtype == THB_F32) {
#pragma unroll
            for (int i = 0; i < GL; i++) f[i] = __uint_as_float(sn[i]);
        } else {
            uint32_t h[GL];
#pragma unroll
            for (int i = 0; i < GL; i++) h[i] = cut.wide ? sn[i / 2] >> (16 * (i & 1)) : sn[i];
            if (p.s_dtype == THB_F16) {
#pragma unroll
                for (int i = 0; i < GL; i++) f[i] = __half2float(__ushort_as_half((unsigned short)h[i]));
            } else {
#pragma unroll
                for (int i = 0; i < GL; i++) f[i] = __uint_as_float(h[i] << 16);
            }
        }
#pragma unroll
        for (int i = 0; i < GL; i++)  // (what lies behind a row's groups is not a scale; rows behind the last have any, and are not written)
            scales[(lane >> 1) * SP + sj + i] = group + i < groups ? f[i] : 0.f;
        if (ZEROS)
#pragma unroll
            for (int i = 0; i < GL; i++) zeros[(lane >> 1) * SP + sj + i] = zero_pair<X::BF>(cut.wide ? zn[i / 4] >> (8 * (i & 3)) : zn[i]);
    };

    // ---- x of a chunk: as loaded, and as operands
    const long xrow = (long)(g < p.N ? g : 0) * p.x_ld;
    const int xk = g < p.N ? p.K : 0;  // (columns beyond the rows of x are zeros)
    XVec<X> raw[NB][4];
    uint32_t xb[NB][4][X::PARTS][4];
    auto x_at = [&](int chunk, int n, int i) { return ((chunk * wk + kw) * cut.mine + n) * 128 + (i / VW) * GROUP + t * 8 * VW + (i % VW) * 8; };
    auto load_x = [&](int chunk) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) raw[n][i].load(p.x, xrow, x_at(chunk, n, i), n < cut.mine ? xk : 0);
    };
    auto take_x = [&](int chunk) {
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int left = p.K - x_at(chunk, n, i);
                if (left > 0 && left < 8) raw[n][i].cut(left);
                raw[n][i].get(xb[n][i]);
            }
    };

    // The weights do not depend on the launch before this one: the first stages are under way while that one drains.
#pragma unroll 1
    for (int u = 0; u < STAGES - 1; u++) fetch();
    fetch_scales(0, tile0 + mw);
    pdl_enter();
    load_x(0);

    // where this lane's codes of row g lie in a stage: pieces differ in bits 4 to 6 by what their number differs in, then by whole lines
    const uint32_t mine_at = warp * STAGES * NB * 1024 + piece(g, t * VW / 4) + t * VW % 4 * 4;
    int slot = 0, parity = 0;
    for (int chunk = 0; chunk < cut.chunks; chunk++) {
        take_x(chunk);
        for (int step = 0; step < steps; step++) {
            __syncwarp();  // (all lanes have read the last unit's)
            put_scales(chunk);
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            fetch();
            const bool last = step == steps - 1;
            fetch_scales(last ? chunk + 1 : chunk, tile0 + mw + (last ? 0 : (step + 1) * wm));
            if (last && chunk + 1 < cut.chunks) load_x(chunk + 1);

            const uint32_t at = mine_at + slot * (NB * 1024);
            slot = slot + 1 == STAGES ? 0 : slot + 1;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            auto block = [&](int n) {
                // the block's scales and zero points of rows g and g + 8
                float sc[2][NG];
                uint32_t zs[2][NG];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int o = (g + 8 * r) * SP + n * NG;
                    if constexpr (NG == 4) {
                        const float4 v = *reinterpret_cast<const float4 *>(scales + o);
                        sc[r][0] = v.x; sc[r][1 % NG] = v.y; sc[r][2 % NG] = v.z; sc[r][3 % NG] = v.w;
                        if (ZEROS) {
                            const uint4 z = *reinterpret_cast<const uint4 *>(zeros + o);
                            zs[r][0] = z.x; zs[r][1 % NG] = z.y; zs[r][2 % NG] = z.z; zs[r][3 % NG] = z.w;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < NG; j++) {
                            sc[r][j] = scales[o + j];
                            if (ZEROS) zs[r][j] = zeros[o + j];
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t w[2][VW], za[2], zb[2];
                    constexpr int LINE = NB >= 2 ? 8 : 4;  // pieces of a row in a line
                    const int c0 = n * 4 + j * (GROUP / 32);
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint8_t *src = smem + (at ^ c0 % LINE * 16) + c0 / LINE * 128 + r * (8 * NB * 64);
                        if constexpr (VW == 4) {
                            const uint4 v = *reinterpret_cast<const uint4 *>(src);
                            w[r][0] = v.x; w[r][1 % VW] = v.y; w[r][2 % VW] = v.z; w[r][3 % VW] = v.w;
                        } else if constexpr (VW == 2) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(src);
                            w[r][0] = v.x; w[r][1 % VW] = v.y;
                        } else
                            w[r][0] = *reinterpret_cast<const uint32_t *>(src);
                        za[r] = ZEROS ? zs[r][j] : zero_pair<X::BF>(8);
                        zb[r] = X::BF ? 0 : zero_pair_16(za[r]);
                    }
#pragma unroll
                    for (int h = 0; h < VW; h++) {
                        uint32_t a[2][4];
#pragma unroll
                        for (int r = 0; r < 2; r++) pairs_of<X::BF>(w[r][h], za[r], zb[r], a[r]);
#pragma unroll
                        for (int q = X::PARTS - 1; q >= 0; q--) {
                            const uint32_t(&b)[4] = xb[n][j * VW + h][q];
                            mma16816<X::BF>(c, a[0][0], a[1][0], a[0][1], a[1][1], b[0], b[1]);
                            mma16816<X::BF>(c, a[0][2], a[1][2], a[0][3], a[1][3], b[2], b[3]);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 4; q++) acc[q] = fmaf(c[q], sc[q >> 1][j], acc[q]);
                }
            };
            if (cut.mine == NB) {  // (without branches between the blocks, whose instructions then overlap)
#pragma unroll
                for (int n = 0; n < NB; n++) block(n);
            } else {
#pragma unroll
                for (int n = 0; n < NB; n++)
                    if (n < cut.mine) block(n);
            }
            // the tile's parts.  c0, c1: row g, columns 2t and 2t + 1; c2, c3: row g + 8
            float *const parts = part + parity * WARPS * PITCH;
#pragma unroll
            for (int q = 0; q < 4; q++) parts[warp * PITCH + (2 * t + (q & 1)) * COL + g + (q >> 1) * 8] = acc[q];
            // Four warps add a tile's parts, two columns each, the other four those of the next tile.  Where a step has one tile, those who
            // do not add only arrive and go on: everybody waits every other step, and what is waited for includes the end of the other
            // four's last addition, so that two buffers are enough, and a tile's sums may pass from four warps to the others.
            const int adding = parity;
            if (wm > 1) __syncthreads();
            else if (warp / 4 == adding) asm volatile("bar.sync %0, %1;" ::"r"(1 + parity), "n"(WARPS * 32) : "memory");
            else asm volatile("bar.arrive %0, %1;" ::"r"(1 + parity), "n"(WARPS * 32) : "memory");
            parity ^= 1;
            for (int i = 0; i < wm; i++) {
                const int turn = wm > 1 ? i & 1 : adding, local = step * wm + i, tile = tile0 + local;
                const int n = (warp & 3) * 2 + (lane >> 4), row = lane & 15, m = tile * 16 + row;
                if (warp / 4 != turn || n >= p.N || tile >= tile1) continue;
                const float *from = parts + i * wk * PITCH + n * COL + row;
                float v = 0.f;
                for (int q = 0; q < wk; q++) v += from[q * PITCH];
                float *sum = sums + local * 128 + n * 16 + row;
                if (chunk > 0) v += *sum;
                if (chunk + 1 < cut.chunks) {
                    *sum = v;
                    continue;
                }
                if (m >= (p.M + 7) / 8 * 8 || (p.dtype == THB_F32 && m >= (p.M + 3) / 4 * 4)) continue;
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
            }
        }
    }
    cp_async_wait<0>();
}

template <typename X, int GROUP, bool ZEROS> int launch_q4_group(const Q4Params &p, cudaStream_t st)
{
    constexpr int NB = Q4Shape<X>::NB, FIXED = Q4Shape<X>::FIXED;
    constexpr int GL = NB * (128 / GROUP) / 2 > 0 ? NB * (128 / GROUP) / 2 : 1;
    const auto kern = gemv_q4_kernel<X, GROUP, ZEROS>;
    static int sms[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_gemv_q4_fwd: device ordinal above 63");
    if (!sms[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FIXED + Q4_ACC * 512);
        if (e != cudaSuccess) return thb_note_launch(e, "gemv_q4_kernel attributes");
        sms[dev] = thb_sm_count();
    }
    Q4Cut c;
    const int blocks = (p.K + 127) / 128;
    c.tiles = (p.M + 15) / 16;
    c.wk = WARPS;
    while (c.wk > 1 && c.wk / 2 * NB >= blocks) c.wk /= 2;
    c.chunks = (blocks + c.wk * NB - 1) / (c.wk * NB);
    c.mine = (blocks + c.wk * c.chunks - 1) / (c.wk * c.chunks);
    c.wide = p.s_dtype != THB_F32 && (c.mine * (128 / GROUP)) % GL == 0 && p.s_ld % GL == 0 && reinterpret_cast<uintptr_t>(p.wscale) % (2 * GL) == 0 &&
             (!p.wzero || (p.z_ld % GL == 0 && reinterpret_cast<uintptr_t>(p.wzero) % GL == 0));
    int grid = c.tiles < sms[dev] ? c.tiles : sms[dev];
    if (c.chunks > 1 && grid < (c.tiles + Q4_ACC - 1) / Q4_ACC) grid = (c.tiles + Q4_ACC - 1) / Q4_ACC;
    const int most = (c.tiles + grid - 1) / grid;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = FIXED + (c.chunks > 1 ? most * 512 : 0);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = thb_pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, c);
    return thb_note_launch(e != cudaSuccess ? e : cudaGetLastError(), "gemv_q4_kernel");
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
