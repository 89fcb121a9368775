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
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// codes i and i + 4 of a word (nibbles, lowest first) less the zero point, as a pair of 16-bit numbers; zp = (zero + base) twice
template <bool BF> __device__ __forceinline__ uint32_t pair_of(uint32_t word, int i, uint32_t zp)
{
    uint32_t v = word >> (4 * i);
    if (BF) {
        v = (v & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&zp));
        return *reinterpret_cast<const uint32_t *>(&d);
    }
    v = (v & 0x000f000fu) | 0x64006400u;
    const __half2 d = __hsub2(*reinterpret_cast<__half2 *>(&v), *reinterpret_cast<const __half2 *>(&zp));
    return *reinterpret_cast<const uint32_t *>(&d);
}

// 8 consecutive values of x from k on as four B registers a part: (x0,x4), (x1,x5), (x2,x6), (x3,x7); zeros from K on
template <typename X> struct XLoad;
template <bool BF16> struct XLoad16 {
    static __device__ __forceinline__ void get(const void *x, long row, int k, int K, uint32_t (&b)[1][4])
    {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < K) {
            v = *reinterpret_cast<const uint4 *>((const uint16_t *)x + row + k);
            if (k + 8 > K) {
                uint32_t *h = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                for (int i = 0; i < 4; i++) h[i] &= k + 2 * i + 1 < K ? 0xffffffffu : k + 2 * i < K ? 0xffffu : 0u;
            }
        }
        b[0][0] = __byte_perm(v.x, v.z, 0x5410);
        b[0][1] = __byte_perm(v.x, v.z, 0x7632);
        b[0][2] = __byte_perm(v.y, v.w, 0x5410);
        b[0][3] = __byte_perm(v.y, v.w, 0x7632);
    }
};
template <> struct XLoad<XF16> : XLoad16<false> {};
template <> struct XLoad<XBF16> : XLoad16<true> {};
template <> struct XLoad<XE4M3> {
    static __device__ __forceinline__ uint32_t two(uint32_t codes)  // two codes in the low halfword -> two fp16
    {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
        return (uint32_t)h.x | (uint32_t)h.y << 16;
    }
    static __device__ __forceinline__ void get(const void *x, long row, int k, int K, uint32_t (&b)[1][4])
    {
        uint2 v = make_uint2(0, 0);
        if (k < K) {
            v = *reinterpret_cast<const uint2 *>((const uint8_t *)x + row + k);
            const int left = K - k;
            if (left < 8) {
                v.x &= left >= 4 ? 0xffffffffu : (1u << 8 * left) - 1;
                v.y &= left <= 4 ? 0u : (1u << 8 * (left - 4)) - 1;
            }
        }
        const uint32_t p = __byte_perm(v.x, v.y, 0x5140), r = __byte_perm(v.x, v.y, 0x7362);  // codes 0 4 1 5 and 2 6 3 7
        b[0][0] = two(p);
        b[0][1] = two(p >> 16);
        b[0][2] = two(r);
        b[0][3] = two(r >> 16);
    }
};
template <> struct XLoad<XF32> {
    static __device__ __forceinline__ void get(const void *x, long row, int k, int K, uint32_t (&b)[3][4])
    {
        float v[8];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            const int at = k + 4 * h;
            if (at < K) {
                f = *reinterpret_cast<const float4 *>((const float *)x + row + at);
                if (at + 1 >= K) f.y = 0.f;
                if (at + 2 >= K) f.z = 0.f;
                if (at + 3 >= K) f.w = 0.f;
            }
            v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
        }
        // a part is the top 16 bits of what the parts before it leave: 8 bits of mantissa each, no rounding, the rest is exact.
        // (infinities and NaN: the first part is the value, the others must not turn an infinity into NaN)
        uint32_t part[3][8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t u = __float_as_uint(v[i]);
            const bool fin = (u & 0x7f800000u) != 0x7f800000u;
            part[0][i] = fin || !(u & 0x7fffffu) ? u : 0x7fc00000u;
            const float r1 = v[i] - __uint_as_float(u & 0xffff0000u);
            part[1][i] = fin ? __float_as_uint(r1) : 0u;
            const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
            part[2][i] = fin ? __float_as_uint(r2) : 0u;
        }
#pragma unroll
        for (int q = 0; q < 3; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) b[q][i] = __byte_perm(part[q][i], part[q][i + 4], 0x7632);
    }
};

__device__ __forceinline__ float wscale_at(const void *s, int dtype, long i)
{
    if (dtype == THB_F32) return ((const float *)s)[i];
    if (dtype == THB_F16) return __half2float(((const __half *)s)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)s)[i]);
}

// A CTA takes 16 rows of weights, its eight warps an eighth of the blocks of 128 k each, in order; the parts are added at the end.
// Lane (g = lane / 4, t = lane % 4) holds rows g and g + 8.  Of a block it loads the k of its t: 32 in one vector where a group is 128
// long, 16 of each of two groups, 8 of each of four, so that a product's k are all of one group.
template <typename X, int GROUP>
__global__ void __launch_bounds__(256) gemv_q4_kernel(Q4Params p)
{
    constexpr int AHEAD = 4;                  // blocks under way a warp
    constexpr int VW = GROUP / 32, NG = 128 / GROUP;  // words a load, groups a block
    __shared__ float part[8][128];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int m0 = blockIdx.x * 16;
    const int blocks = (p.K + 127) / 128, groups = (p.K + GROUP - 1) / GROUP, bytes = ((p.K + 1) / 2 + 15) / 16 * 16;
    const int b0 = blocks * warp / 8, b1 = blocks * (warp + 1) / 8;
    // (rows beyond the last are read as the last and not written)
    const long row[2] = {min(m0 + g, p.M - 1), min(m0 + g + 8, p.M - 1)};

    uint32_t w[AHEAD][2][4];
    float s[AHEAD][2][NG];
    uint32_t z[AHEAD][2][NG];
    auto load = [&](int slot, int b) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const uint8_t *at = p.w + row[r] * p.w_ld;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const int o = b * 64 + j * (GROUP / 2) + t * 4 * VW;
                uint32_t *d = w[slot][r] + j * VW;
#pragma unroll
                for (int i = 0; i < VW; i++) d[i] = 0;
                s[slot][r][j] = 0.f;
                z[slot][r][j] = 8;
                if (b < b1 && o < bytes) {
                    if (VW == 4) {
                        const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(at + o));
                        d[0] = v.x; d[1 % VW] = v.y; d[2 % VW] = v.z; d[3 % VW] = v.w;
                    } else if (VW == 2) {
                        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(at + o));
                        d[0] = v.x; d[1 % VW] = v.y;
                    } else
                        d[0] = __ldg(reinterpret_cast<const uint32_t *>(at + o));
                }
                const int group = b * NG + j;
                if (b < b1 && group < groups) {
                    s[slot][r][j] = wscale_at(p.wscale, p.s_dtype, row[r] * p.s_ld + group);
                    if (p.wzero) z[slot][r][j] = p.wzero[row[r] * p.z_ld + group];
                }
            }
        }
    };
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    const long xrow = (long)(g < p.N ? g : 0) * p.x_ld;
    const int xk = g < p.N ? p.K : 0;  // (columns beyond the rows of x are zeros)
    auto consume = [&](int slot, int b) {
#pragma unroll
        for (int j = 0; j < NG; j++) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t zp[2];
#pragma unroll
            for (int r = 0; r < 2; r++) zp[r] = ((z[slot][r][j] & 15) | (X::BF ? 0x4300u : 0x6400u)) * 0x10001u;
#pragma unroll
            for (int i = 0; i < VW; i++) {
                uint32_t xb[X::PARTS][4];
                XLoad<X>::get(p.x, xrow, b * 128 + j * GROUP + t * 8 * VW + i * 8, xk, xb);
                uint32_t a[2][4];
#pragma unroll
                for (int r = 0; r < 2; r++)
#pragma unroll
                    for (int q = 0; q < 4; q++) a[r][q] = pair_of<X::BF>(w[slot][r][j * VW + i], q, zp[r]);
#pragma unroll
                for (int q = X::PARTS - 1; q >= 0; q--) {
                    mma16816<X::BF>(c, a[0][0], a[1][0], a[0][1], a[1][1], xb[q][0], xb[q][1]);
                    mma16816<X::BF>(c, a[0][2], a[1][2], a[0][3], a[1][3], xb[q][2], xb[q][3]);
                }
            }
            acc[0] = fmaf(c[0], s[slot][0][j], acc[0]);
            acc[1] = fmaf(c[1], s[slot][0][j], acc[1]);
            acc[2] = fmaf(c[2], s[slot][1][j], acc[2]);
            acc[3] = fmaf(c[3], s[slot][1][j], acc[3]);
        }
    };
    // The weights do not depend on the launch before this one: the first blocks are under way while that one drains.
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(i, b0 + i);
    pdl_enter();
    for (int b = b0; b < b1; b += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (b + i >= b1) break;
            consume(i, b + i);
            load(i, b + i + AHEAD);
        }
    }
    // c0, c1: row g, columns 2t and 2t + 1; c2, c3: row g + 8
#pragma unroll
    for (int i = 0; i < 4; i++) part[warp][(2 * t + (i & 1)) * 16 + g + (i >> 1) * 8] = acc[i];
    __syncthreads();
    if (tid < 128) {
        const int n = tid >> 4, m = m0 + (tid & 15);
        const int al = p.dtype == THB_F32 ? 4 : 8;
        if (n < p.N && m < p.M) {
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < 8; q++) v += part[q][tid];
            if (p.x_scale) v *= p.x_scale[n];
            const float sc = p.scale ? p.scale[m] : 1.f, sh = p.shift ? p.shift[m] : 0.f;
            const float sl = p.act.kind == THB_ACT_PRELU ? p.act.slope[m] : 0.f;
            v = thb_apply_act(v * sc + sh, p.act.kind, p.act.threshold, p.act.value, p.act.alpha, sl);
            const long o = (long)n * p.y_ld + m;
            if (p.dtype == THB_F32) ((float *)p.y)[o] = v;
            else if (p.dtype == THB_F16) ((__half *)p.y)[o] = __float2half_rn(v);
            else ((__nv_bfloat16 *)p.y)[o] = __float2bfloat16_rn(v);
        } else if (n < p.N && m < (p.M + al - 1) / al * al) {
            // channels of the padded tail of y are kept at exact zero
            const long o = (long)n * p.y_ld + m;
            if (p.dtype == THB_F32) ((float *)p.y)[o] = 0.f;
            else ((uint16_t *)p.y)[o] = 0;
        }
    }
}

template <typename X> int launch_q4(const Q4Params &p, int group, cudaStream_t st)
{
    const unsigned grid = (p.M + 15) / 16;
    switch (group) {
    case 32: thb_launch(gemv_q4_kernel<X, 32>, grid, 256, st, p); break;
    case 64: thb_launch(gemv_q4_kernel<X, 64>, grid, 256, st, p); break;
    default: thb_launch(gemv_q4_kernel<X, 128>, grid, 256, st, p);
    }
    return THB_LAUNCH_CHECK("gemv_q4_kernel");
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
