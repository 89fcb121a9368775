// Root-mean-square norm with the residual's addition and an optional result in e4m3 with a scale a row.
//     t = x + res;  v = t * r * gain, r = 1/sqrt(mean(t^2) + eps);  q = e4m3(v / (max|v| / 448))
// One pass: a row's t stay in registers between the reduction and the results.  r is common to a row, so max|v| = r * max|t * gain|
// and the codes are e4m3(t * gain * (448 / max|t * gain|)): the sum of squares and the maximum are reduced together, and r's
// rounding does not reach the codes.  HBM-bound on many rows, latency-bound on few.
#include "tokens.cuh"
#include <cuda_fp8.h>

namespace {

struct NormParams {
    const void *x, *res;
    void *sum, *y;
    uint8_t *q;
    float *q_scale;
    const float *gain;
    long rows;
    int C, x_ld, res_ld, sum_ld, y_ld, q_ld;
    float eps;
};

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// WARP: groups of `lanes` threads (a power of two up to a warp) have a row each; otherwise the whole block shares one.
// A thread owns vectors tid, tid + threads, ... of its row, VPT at most.  Short rows (VPT <= 2) have the next row under way while
// one is reduced and written, and keep the gain in registers where there is one vector of it; long ones fill the SM by themselves.
template <typename T, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512) rmsnorm_kernel(NormParams p, int lanes)
{
    constexpr int VN = Vec16<T>::N;
    constexpr bool AHEAD = VPT <= 2, KEEP = VPT == 1;
    __shared__ float2 part[2][32];
    pdl_enter();
    const int threads = WARP ? lanes : blockDim.x, tid = WARP ? threadIdx.x % lanes : threadIdx.x;
    const int per_block = WARP ? blockDim.x / lanes : 1;
    const long first = (long)blockIdx.x * per_block + (WARP ? threadIdx.x / lanes : 0), step = (long)gridDim.x * per_block;
    const int nv = (p.C + VN - 1) / VN, nvq = (p.C + 15) / 16 * (16 / VN);  // (8-bit rows are padded to 16 values)

    auto gain_of = [&](int v, float *g) {
#pragma unroll
        for (int j = 0; j < VN; j++) g[j] = p.gain && v * VN + j < p.C ? p.gain[v * VN + j] : 1.f;
    };
    float kept[VN];
    if (KEEP) gain_of(tid, kept);

    uint4 xb[VPT], rb[VPT];
    auto load = [&](long row) {
        if (row >= p.rows) return;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int v = tid + i * threads;
            if (v < nv) {
                xb[i] = *reinterpret_cast<const uint4 *>((const T *)p.x + row * p.x_ld + (long)v * VN);
                if (p.res) rb[i] = *reinterpret_cast<const uint4 *>((const T *)p.res + row * p.res_ld + (long)v * VN);
            }
        }
    };
    if (AHEAD) load(first);
    int parity = 0;
    // (all threads of a warp take the same number of turns: the reductions name whole warps)
    const long block_first = (long)blockIdx.x * per_block;
    for (long base = block_first; base < p.rows; base += step) {
        const long row = base + (first - block_first);
        const bool live = row < p.rows;
        float t[VPT][VN], square = 0.f, most = 0.f;
        if (!AHEAD) load(row);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int v = tid + i * threads;
            if (live && v < nv) {
                Vec16<T>::unpack(xb[i], t[i]);
                if (p.res) {
                    float r[VN];
                    Vec16<T>::unpack(rb[i], r);
#pragma unroll
                    for (int j = 0; j < VN; j++) t[i][j] += r[j];
                }
                float g[VN];
                if (!KEEP && p.q) gain_of(v, g);
#pragma unroll
                for (int j = 0; j < VN; j++) {
                    if (v * VN + j >= p.C) t[i][j] = 0.f;
                    square = fmaf(t[i][j], t[i][j], square);
                    if (p.q) most = max_nan(most, fabsf(t[i][j] * (KEEP ? kept[j] : g[j])));
                }
                if (p.sum) *reinterpret_cast<uint4 *>((T *)p.sum + row * p.sum_ld + (long)v * VN) = Vec16<T>::pack(t[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VN; j++) t[i][j] = 0.f;
            }
        }
        if (AHEAD) load(row + step);
        const int width = WARP ? lanes : 32;
        for (int o = width / 2; o > 0; o >>= 1) {
            square += __shfl_xor_sync(0xffffffffu, square, o);
            most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        if (!WARP) {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
            if (lane == 0) part[parity][warp] = make_float2(square, most);
            __syncthreads();
            const float2 o = lane < warps ? part[parity][lane] : make_float2(0.f, 0.f);
            square = o.x;
            most = o.y;
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) {
                square += __shfl_xor_sync(0xffffffffu, square, k);
                most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, k));
            }
            parity ^= 1;  // (the buffers alternate, so that one barrier a row is enough)
        }
        const float r = rsqrtf(square / (float)p.C + p.eps);
        float scale = 0.f, code = 0.f;
        if (p.q) {
            const float top = r * most;
            if (!isfinite(square) || !isfinite(top)) scale = __int_as_float(0x7fc00000);
            else if (top >= 0x1p-100f) {
                scale = top / 448.f;
                code = 448.f / most;
            }
            if (live && tid == 0) p.q_scale[row] = scale;
        }
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int v = tid + i * threads;
            float g[VN];
            if (!KEEP) gain_of(v, g);
            if (p.q && v < nvq) {
                uint32_t c[VN / 4];
#pragma unroll
                for (int j = 0; j < VN; j += 4) {
                    float w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = t[i][j + k] * (KEEP ? kept[j + k] : g[j + k]) * code;
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(w[0], w[1]), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(w[2], w[3]), __NV_SATFINITE, __NV_E4M3);
                    c[j / 4] = lo | hi << 16;
                }
                uint8_t *at = p.q + row * p.q_ld + (long)v * VN;
                if (VN == 4) *reinterpret_cast<uint32_t *>(at) = c[0];
                else *reinterpret_cast<uint2 *>(at) = make_uint2(c[0], c[VN / 4 - 1]);
            }
            if (p.y && v < nv) {
                float w[VN];
#pragma unroll
                for (int j = 0; j < VN; j++) w[j] = v * VN + j < p.C ? t[i][j] * r * (KEEP ? kept[j] : g[j]) : 0.f;
                *reinterpret_cast<uint4 *>((T *)p.y + row * p.y_ld + (long)v * VN) = Vec16<T>::pack(w);
            }
        }
    }
}

template <typename T> int launch_rmsnorm(const NormParams &p, cudaStream_t st)
{
    constexpr int VN = Vec16<T>::N;
    const int nv = (p.C + 15) / 16 * (16 / VN), sms = thb_sm_count();
    if (nv <= 32) {
        int lanes = 1;
        while (lanes < nv) lanes *= 2;
        const long blocks = (p.rows + 256 / lanes - 1) / (256 / lanes);
        thb_launch(rmsnorm_kernel<T, 1, true>, (unsigned)(blocks < 8 * sms ? blocks : 8 * sms), 256, st, p, lanes);
        return THB_LAUNCH_CHECK("rmsnorm_kernel");
    }
    const int vpt = nv <= 512 ? 1 : nv <= 1024 ? 2 : nv <= 2048 ? 4 : nv <= 4096 ? 8 : 16;
    const int threads = ((nv + vpt - 1) / vpt + 31) / 32 * 32, resident = 2048 / threads;
    const unsigned grid = (unsigned)(p.rows < (long)resident * sms ? p.rows : (long)resident * sms);
    switch (vpt) {
    case 1: thb_launch(rmsnorm_kernel<T, 1, false>, grid, threads, st, p, 0); break;
    case 2: thb_launch(rmsnorm_kernel<T, 2, false>, grid, threads, st, p, 0); break;
    case 4: thb_launch(rmsnorm_kernel<T, 4, false>, grid, threads, st, p, 0); break;
    case 8: thb_launch(rmsnorm_kernel<T, 8, false>, grid, threads, st, p, 0); break;
    default:
        if constexpr (VN == 4) thb_launch(rmsnorm_kernel<T, 16, false>, grid, threads, st, p, 0);  // (only rows of fp32 are this many vectors)
    }
    return THB_LAUNCH_CHECK("rmsnorm_kernel");
}

}  // namespace

extern "C" int thb_rmsnorm_fwd(const thb_rmsnorm_desc *d, const void *x, const void *res, void *sum, void *y, void *q, float *q_scale,
                               thb_stream s)
{
    if (!d) return THB_ERR_ARG;
    if (d->dtype != THB_F32 && d->dtype != THB_F16 && d->dtype != THB_BF16)
        return thb_refuse(THB_ERR_UNSUPPORTED, "thb_rmsnorm_fwd: dtype is not THB_F32, THB_F16 or THB_BF16");
    if (d->rows < 0 || d->C < 1 || !(d->eps >= 0.f)) return thb_refuse(THB_ERR_ARG, "thb_rmsnorm_fwd: rows < 0, C < 1 or eps < 0");
    if (d->C > 32768) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_rmsnorm_fwd: rows of more than 32768 values");
    if (d->rows == 0) return THB_OK;
    if (!x || (!sum && !y && !q) || !q != !q_scale)
        return thb_refuse(THB_ERR_ARG, "thb_rmsnorm_fwd: x, one of sum, y and q, and q_scale with q must be set");
    const int al = thb_channel_align(d->dtype);
    const struct { const void *p; int ld, al; } t[] = {{x, d->x_ld, al}, {res, d->res_ld, al}, {sum, d->sum_ld, al}, {y, d->y_ld, al}, {q, d->q_ld, 16}};
    for (const auto &e : t)
        if (e.p && (thb_misaligned(e.p) || e.ld % e.al || e.ld < d->C))
            return thb_refuse(THB_ERR_ARG, "thb_rmsnorm_fwd: a tensor is not 16-byte aligned, or its ld is below C or no multiple of the alignment");
    const NormParams p = {x, res, sum, y, (uint8_t *)q, q_scale, d->gain, d->rows, d->C, d->x_ld, d->res_ld, d->sum_ld, d->y_ld, d->q_ld, d->eps};
    switch (d->dtype) {
    case THB_F32: return launch_rmsnorm<float>(p, (cudaStream_t)s);
    case THB_F16: return launch_rmsnorm<__half>(p, (cudaStream_t)s);
    default: return launch_rmsnorm<__nv_bfloat16>(p, (cudaStream_t)s);
    }
}
