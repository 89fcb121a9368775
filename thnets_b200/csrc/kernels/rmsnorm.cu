// Root-mean-square norm with the residual's addition and an optional result in e4m3 with a scale a row.
//     t = x + res;  v = t * r * gain, r = 1/sqrt(mean(t^2) + eps);  q = e4m3(v / (max|v| / 448))
// One pass: a row's t stay in registers between the reduction and the results.  r is common to a row, so max|v| = r * max|t * gain|
// and the codes are e4m3(t * gain * (448 / max|t * gain|)): the sum of squares and the maximum are reduced together, and r's
// rounding does not reach the codes.  HBM-bound on many rows, and near it by the instructions a value takes; latency-bound on few.
// us a launch in a chain (share of the measured copy rate): 8192 rows of 4096 in fp16 with residual 43.3 (95 %), without residual 26.9 (76 %);
// 4096 of 8192 42.8 (96 %); 2048 of 16384 60 (68 %); 262144 of 128 30.6 (67 %); 8192 of 4096 in fp32 90 (91 %).  To e4m3, whose codes are
// settled as below: 8192 of 4096 in bf16 with residual 49.8 (72 %; 41.1 with codes that the roundings of fp32 decide), y besides 56.2 (82 %, 57.5),
// fp32 81.5 (82 %, 76.9), bf16 without residual 41.3 (37 %, 33.2), 262144 of 128 without 41.3 (38 %, 32.0), 30000 of 1000 in fp16 53 (61 %, 42),
// 4096 of 8192 61 (58 %, 41), 2048 of 16384 79 (45 %, 55), 1024 of 32768 in fp32 162 (42 %, 138).
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

// Codes are what the formula gives in exact arithmetic, rounded to fp32 and that to e4m3.  t * gain * (448 / max) in fp32 is off by 7 units of
// 2^-24 of itself at most (t, its product, the maximum (two), the quotient, EDGE's product, the last one), EDGE is eight: where the codes
// of a little less and of a little more agree they are the code.  For the others, one value in a hundred thousand, fp64 leaves t's and the
// maximum's roundings (three units; without a residual one, the maximum's); what that does not settle takes the row's maximum in exact
// arithmetic, for which its threads come together once more.  Half of what it costs is the instructions of every row and the barrier that asks
// whether any code is open, half the rows with such a value, 1 to 3 us each, of which one CTA has more than the others.  Tried and slower
// (8192 of 4096 in bf16, four blocks an SM, 58.6 us): the exact maximum of every row ahead of its first barrier 66 us; all that is rare out of line
// 124 (its calls spill the row's registers); x and res kept in the ring until the row is done 68; rows with such values left for the end of the launch
// 61 (16384: 125).
constexpr float EDGE = 8 * 0x1p-24f;
// below this maximum 448 / max or the products leave fp32's range: all of the row's codes are settled in fp64
constexpr float LEAST = 0x1p-100f;

__device__ __forceinline__ uint32_t e4m3_of(double v) { return __nv_cvt_float_to_fp8((float)v, __NV_SATFINITE, __NV_E4M3); }

// WARP: groups of `lanes` threads (a power of two up to a warp) have a row each; otherwise the whole block shares one.
// A thread owns vectors tid, tid + threads, ... of its row, VPT at most.  Blocks stay for many rows.  Q: codes are wanted, and with them
// the row's maximum.
// What a block reads next is under way while a row is reduced and written: short rows' vectors in registers, longer ones' in a ring of
// STAGES rows in shared memory by cp.async, of which every thread reads only what it asked for itself, so that nobody waits for another.
// The gain is in registers where a thread has one or two vectors of it, else in shared memory where that has room.
template <typename T, int VPT, bool WARP> struct NormShape {
    static constexpr int VN = Vec16<T>::N;
    static constexpr int STAGES = WARP ? 0 : VPT <= 4 ? 2 : VPT == 8 ? 1 : 0;
    static constexpr bool KEEP = VPT <= 2, GLOBAL = VPT == 8 && VN == 8;
    static int smem(int threads, int nvq, bool res)
    {
        return STAGES * VPT * threads * 16 * (res ? 2 : 1) + (KEEP || GLOBAL ? 0 : nvq * VN * 4);
    }
};
// MOST: threads a block at most.  With codes the registers decide how many blocks stay on an SM: rows of two vectors for each of 256 threads take 80
// and three blocks (8192 rows of 4096 in bf16 with residual: 49.7 us; in 64, which spill, and four 58.6), of up to 512 threads 64 and two (4096
// rows of 8192: 61.2; four vectors for each of 256 threads 71.1), one vector a thread 64.
template <typename T, int VPT, bool WARP, bool Q, int MOST>
__global__ void __launch_bounds__(MOST, !Q ? 0 : WARP || VPT == 1 ? 1024 / MOST : VPT == 2 ? (MOST == 256 ? 3 : 2) : 1) rmsnorm_kernel(NormParams p, int lanes)
{
    using S = NormShape<T, VPT, WARP>;
    constexpr int VN = S::VN, STAGES = S::STAGES;
    constexpr bool KEEP = S::KEEP;
    __shared__ float2 part[2][16];
    __shared__ unsigned long long largest;
    extern __shared__ uint4 smem[];
    const int threads = WARP ? lanes : blockDim.x, tid = WARP ? threadIdx.x % lanes : threadIdx.x;
    const int per_block = WARP ? blockDim.x / lanes : 1;
    const int nv = (p.C + VN - 1) / VN, nvq = (p.C + 15) / 16 * (16 / VN);  // (8-bit rows are padded to 16 values)
    const int slot_size = VPT * threads * (p.res ? 2 : 1);                  // vectors a stage: x's, then those of res
    float4 *const gains = reinterpret_cast<float4 *>(smem + STAGES * slot_size);
    pdl_enter();

    const long base0 = (long)blockIdx.x * per_block, step = (long)gridDim.x * per_block;
    const int sub = WARP ? threadIdx.x / lanes : 0;
    auto stage = [&](int slot, long row) {  // this thread's vectors of a row into its places of the ring
        if (row < p.rows)
#pragma unroll
            for (int i = 0; i < VPT; i++) {
                const int v = tid + i * threads;
                if (v < nv) {
                    cp_async16(smem_u32(smem + slot * slot_size + v), (const T *)p.x + row * p.x_ld + v * VN, 16);
                    if (p.res) cp_async16(smem_u32(smem + slot * slot_size + VPT * threads + v), (const T *)p.res + row * p.res_ld + v * VN, 16);
                }
            }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES; i++) stage(i, base0 + i * step);

    float kept[KEEP ? VPT : 1][VN];
    if (KEEP) {
#pragma unroll
        for (int i = 0; i < (KEEP ? VPT : 1); i++)
#pragma unroll
            for (int j = 0; j < VN; j++) {
                const int c = (tid + i * threads) * VN + j;
                kept[i][j] = p.gain && c < p.C ? p.gain[c] : 1.f;
            }
    } else if (!S::GLOBAL) {
        for (int c = threadIdx.x; c < nvq * VN; c += blockDim.x) reinterpret_cast<float *>(gains)[c] = p.gain && c < p.C ? p.gain[c] : 1.f;
        __syncthreads();
    }
    auto gain_of = [&](int i, int v, float (&g)[VN]) {
        if constexpr (KEEP) {
#pragma unroll
            for (int j = 0; j < VN; j++) g[j] = kept[KEEP ? i : 0][j];
        } else if constexpr (S::GLOBAL) {
#pragma unroll
            for (int j = 0; j < VN; j++) g[j] = p.gain && v * VN + j < p.C ? p.gain[v * VN + j] : 1.f;
        } else {
#pragma unroll
            for (int j = 0; j < VN / 4; j++) {
                const float4 f = gains[v * (VN / 4) + j];
                g[4 * j] = f.x; g[4 * j + 1] = f.y; g[4 * j + 2] = f.z; g[4 * j + 3] = f.w;
            }
        }
    };

    uint4 xb = make_uint4(0, 0, 0, 0), rb = xb;
    auto load = [&](long row) {  // (short rows: one vector a thread)
        if (row < p.rows && tid < nv) {
            xb = *reinterpret_cast<const uint4 *>((const T *)p.x + row * p.x_ld + tid * VN);
            if (p.res) rb = *reinterpret_cast<const uint4 *>((const T *)p.res + row * p.res_ld + tid * VN);
        }
    };
    // (all threads of a block take the same number of turns: the reductions name whole warps)
    const float inv_c = 1.f / (float)p.C;
    if (WARP) load(base0 + sub);
    int parity = 0, slot = 0;
    for (long base = base0; base < p.rows; base += step) {
        const long row = base + sub;
        const bool live = row < p.rows;
        float t[VPT][VN], square = 0.f, most = 0.f;
        if (STAGES > 0) cp_async_wait<STAGES - 1 < 0 ? 0 : STAGES - 1>();
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int v = tid + i * threads;
            if (live && v < nv) {
                if (STAGES > 0) xb = smem[slot * slot_size + v];
                else if (!WARP) xb = *reinterpret_cast<const uint4 *>((const T *)p.x + row * p.x_ld + v * VN);
                Vec16<T>::unpack(xb, t[i]);
                if (p.res) {
                    float r[VN];
                    if (STAGES > 0) rb = smem[slot * slot_size + VPT * threads + v];
                    else if (!WARP) rb = *reinterpret_cast<const uint4 *>((const T *)p.res + row * p.res_ld + v * VN);
                    Vec16<T>::unpack(rb, r);
#pragma unroll
                    for (int j = 0; j < VN; j++) t[i][j] += r[j];
                }
                if ((v + 1) * VN > p.C)
#pragma unroll
                    for (int j = 0; j < VN; j++)
                        if (v * VN + j >= p.C) t[i][j] = 0.f;
#pragma unroll
                for (int j = 0; j < VN; j++) square = fmaf(t[i][j], t[i][j], square);
                if (Q) {
                    float g[VN];
                    gain_of(i, v, g);
#pragma unroll
                    for (int j = 0; j < VN; j++) most = max_nan(most, fabsf(t[i][j] * g[j]));
                }
                if (!Q && p.sum) *reinterpret_cast<uint4 *>((T *)p.sum + row * p.sum_ld + v * VN) = Vec16<T>::pack(t[i]);
            } else {
#pragma unroll
                for (int j = 0; j < VN; j++) t[i][j] = 0.f;
            }
        }
        if (WARP) load(row + step);
        if (STAGES > 0) {
            stage(slot, base + STAGES * step);
            slot = slot + 1 == STAGES ? 0 : slot + 1;
        }
        const int width = WARP ? lanes : 32;
        const float own = most;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            if (o >= width) continue;
            square += __shfl_xor_sync(0xffffffffu, square, o);
            if (Q) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        if (!WARP) {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
            if (lane == 0) part[parity][warp] = make_float2(square, most);
            __syncthreads();
            const float2 o = lane < warps ? part[parity][lane & 15] : make_float2(0.f, 0.f);
            square = o.x;
            most = o.y;
#pragma unroll
            for (int k = 16; k > 0; k >>= 1) {
                square += __shfl_xor_sync(0xffffffffu, square, k);
                if (Q) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, k));
            }
            parity ^= 1;  // (the buffers alternate, so that one barrier a row is enough)
        }
        const float r = rsqrtf(square * inv_c + p.eps);
        if (Q) {
            float scale = 0.f, code = 0.f;
            bool all = false;
            const float top = r * most;
            if (!isfinite(square) || !isfinite(top)) scale = __int_as_float(0x7fc00000);
            else if (top >= 0x1p-100f) {
                scale = top / 448.f;
                all = most < LEAST;
                if (!all) code = 448.f / most;
            }
            if (live && tid == 0) p.q_scale[row] = scale;
            const float up = code * (1.f + EDGE), down = code * (1.f - EDGE);
            unsigned long long marks = 0;  // of this thread's values: those that are not settled
#pragma unroll
            for (int i = 0; i < VPT; i++) {
                const int v = tid + i * threads;
                if (!live || v >= nvq) continue;
                float g[VN];
                gain_of(i, v, g);
                uint32_t c[VN / 4], differs[VN / 4], apart = 0;
#pragma unroll
                for (int j = 0; j < VN; j += 4) {
                    float w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = t[i][j + k] * g[j + k];
                    auto codes = [&](float by) {
                        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(w[0] * by, w[1] * by), __NV_SATFINITE, __NV_E4M3);
                        return lo | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(w[2] * by, w[3] * by), __NV_SATFINITE, __NV_E4M3) << 16;
                    };
                    c[j / 4] = codes(up);
                    apart |= differs[j / 4] = c[j / 4] ^ codes(down);
                }
                uint8_t *at = p.q + row * p.q_ld + v * VN;
                if (VN == 4) *reinterpret_cast<uint32_t *>(at) = c[0];
                else *reinterpret_cast<uint2 *>(at) = make_uint2(c[0], c[VN / 4 - 1]);
                if (apart || all)
#pragma unroll
                    for (int j = 0; j < VN; j++)
                        if (v * VN + j < p.C && (all || differs[j / 4] >> 8 * (j % 4) & 0xff)) marks |= 1ull << (i * VN + j);
            }
            // one marked value after the other (most often there is one): `settled` stores its code or leaves it
            auto each = [&](unsigned long long left, auto settled) {
#pragma unroll 1
                for (; left; left &= left - 1) {
                    const int at = __ffsll((long long)left) - 1, e = (tid + at / VN * threads) * VN + at % VN;
                    if (settled(at, e, p.gain ? p.gain[e] : 1.f)) marks &= ~(1ull << at);
                }
            };
            if (marks && !all) {
                const double by = (double)code + (448. - (double)code * (double)most) * ((double)code * (1. / 448.)), off = (p.res ? 3.01 : 1.01) * 0x1p-24;
                each(marks, [&](int at, int e, float g) {
                    float a = 0.f;
#pragma unroll
                    for (int i = 0; i < VPT * VN; i++) a = i == at ? t[i / VN][i % VN] : a;
                    const double w = (double)a * (double)g * by;
                    const uint32_t q = e4m3_of(w * (1. + off));
                    if (q != e4m3_of(w * (1. - off))) return false;
                    p.q[row * p.q_ld + e] = (uint8_t)q;
                    return true;
                });
            }
            bool any;
            if (WARP) any = __any_sync(0xffffffffu, marks != 0);
            else {
                if (tid == 0) largest = 0;  // (who read it for the row before has passed this row's first barrier since)
                any = __syncthreads_or(marks != 0);
            }
            if (any) {
                // (sum and y, which may take the place of x and res, are not written yet)
                auto exact_of = [&](int e, float g) {
                    const double x = dt<T>::ld((const T *)p.x + row * p.x_ld + e), res = p.res ? dt<T>::ld((const T *)p.res + row * p.res_ld + e) : 0.f;
                    return (x + res) * (double)g;
                };
                // the row's largest is among those within EDGE of fp32's
                const float least = most < LEAST ? 0.f : most * (1.f - EDGE);
                double exact = 0.;
                if (live && own >= least) {
                    unsigned long long near = 0;
#pragma unroll
                    for (int i = 0; i < VPT; i++) {
                        const int v = tid + i * threads;
                        float g[VN];
                        if (v >= nv) continue;
                        gain_of(i, v, g);
#pragma unroll
                        for (int j = 0; j < VN; j++)
                            if (v * VN + j < p.C && fabsf(t[i][j] * g[j]) >= least) near |= 1ull << (i * VN + j);
                    }
                    each(near, [&](int, int e, float g) {
                        exact = fmax(exact, fabs(exact_of(e, g)));
                        return false;
                    });
                }
                if (WARP) {
                    for (int o = lanes / 2; o > 0; o >>= 1) exact = fmax(exact, __shfl_xor_sync(0xffffffffu, exact, o));
                } else {
                    if (exact > 0.) atomicMax(&largest, (unsigned long long)__double_as_longlong(exact));  // (doubles above zero are in the order of their bits)
                    __syncthreads();
                    exact = __longlong_as_double((long long)largest);
                }
                if (all && tid == 0 && live) p.q_scale[row] = (float)((double)r * (exact / 448.));
                if (marks) {
                    exact = 448. / exact;
                    each(marks, [&](int, int e, float g) {
                        p.q[row * p.q_ld + e] = (uint8_t)e4m3_of(exact_of(e, g) * exact);
                        return true;
                    });
                }
            }
        }
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int v = tid + i * threads;
            if (v >= nv) continue;
            float g[VN], w[VN];
            gain_of(i, v, g);
            if (Q && p.sum) *reinterpret_cast<uint4 *>((T *)p.sum + row * p.sum_ld + v * VN) = Vec16<T>::pack(t[i]);
            if (p.y) {
#pragma unroll
                for (int j = 0; j < VN; j++) w[j] = t[i][j] * r * g[j];
                if ((v + 1) * VN > p.C)  // (zeros behind the row, whatever r is)
#pragma unroll
                    for (int j = 0; j < VN; j++)
                        if (v * VN + j >= p.C) w[j] = 0.f;
                *reinterpret_cast<uint4 *>((T *)p.y + row * p.y_ld + v * VN) = Vec16<T>::pack(w);
            }
        }
    }
}

template <typename T, int VPT, bool Q, int MOST = 512> int launch_block(const NormParams &p, cudaStream_t st)
{
    using S = NormShape<T, VPT, false>;
    const auto kern = rmsnorm_kernel<T, VPT, false, Q, MOST>;
    const int nvq = (p.C + 15) / 16 * (16 / S::VN), threads = ((nvq + VPT - 1) / VPT + 31) / 32 * 32, smem = S::smem(threads, nvq, p.res != nullptr);
    static int sms[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return thb_refuse(THB_ERR_UNSUPPORTED, "thb_rmsnorm_fwd: device ordinal above 63");
    if (!sms[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return thb_note_launch(e, "rmsnorm_kernel attributes");
        sms[dev] = thb_sm_count();
    }
    // As many blocks as stay on the device at once, each with many rows: with two vectors a thread so many that 64 KB are under way an SM
    // (8192 rows of 4096 in 16 bits with a residual: 43.6 us with two blocks of 256 threads, 52.8 with four; without one 30.5 and 26.9), with one
    // as many as there is room for (30000 rows of 1000: 48.7 us with 1024 threads an SM, 40.8 with 2048).
    const int by_smem = 220 * 1024 / (smem + 2048), by_threads = (VPT == 1 ? 2048 : VPT == 2 && Q ? (MOST == 256 ? 768 : 1024) : VPT == 2 && !p.res ? 1024 : 512) / threads, resident = by_smem < by_threads ? by_smem : by_threads;
    const long most = (long)(resident < 1 ? 1 : resident) * sms[dev];
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.rows < most ? p.rows : most));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = thb_pdl_enabled() ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, 0);
    return thb_note_launch(e != cudaSuccess ? e : cudaGetLastError(), "rmsnorm_kernel");
}

template <typename T, bool Q> int launch_rmsnorm(const NormParams &p, cudaStream_t st)
{
    constexpr int VN = Vec16<T>::N;
    const int nv = (p.C + 15) / 16 * (16 / VN);
    if (nv <= 32) {
        int lanes = 1;
        while (lanes < nv) lanes *= 2;
        const long blocks = (p.rows + 256 / lanes - 1) / (256 / lanes), most = 8L * thb_sm_count();
        thb_launch(rmsnorm_kernel<T, 1, true, Q, 256>, (unsigned)(blocks < most ? blocks : most), 256, st, p, lanes);
        return THB_LAUNCH_CHECK("rmsnorm_kernel");
    }
    if (nv <= 256) return launch_block<T, 1, Q, 256>(p, st);
    if constexpr (Q)
        if (nv <= 512) return launch_block<T, 2, Q, 256>(p, st);
    if (nv <= 1024) return launch_block<T, 2, Q>(p, st);
    if (nv <= 2048) return launch_block<T, 4, Q>(p, st);
    if (nv <= 4096) return launch_block<T, 8, Q>(p, st);
    if constexpr (VN == 4) return launch_block<T, 16, Q>(p, st);  // (only rows of fp32 are this many vectors)
    return THB_ERR_UNSUPPORTED;
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
    // in place row by row only, and no two results in one place
    auto moved = [&](const void *out, int ld) { return out && d->rows > 1 && ((out == x && ld != d->x_ld) || (out == res && ld != d->res_ld)); };
    if (moved(sum, d->sum_ld) || moved(y, d->y_ld) || (sum && sum == y) || (q && (q == x || q == res || q == sum || q == y)))
        return thb_refuse(THB_ERR_ARG, "thb_rmsnorm_fwd: a result in the place of an input with another ld, two results in one place, or q in the place of another tensor");
    const NormParams p = {x, res, sum, y, (uint8_t *)q, q_scale, d->gain, d->rows, d->C, d->x_ld, d->res_ld, d->sum_ld, d->y_ld, d->q_ld, d->eps};
    switch (d->dtype) {
    case THB_F32: return q ? launch_rmsnorm<float, true>(p, (cudaStream_t)s) : launch_rmsnorm<float, false>(p, (cudaStream_t)s);
    case THB_F16: return q ? launch_rmsnorm<__half, true>(p, (cudaStream_t)s) : launch_rmsnorm<__half, false>(p, (cudaStream_t)s);
    default: return q ? launch_rmsnorm<__nv_bfloat16, true>(p, (cudaStream_t)s) : launch_rmsnorm<__nv_bfloat16, false>(p, (cudaStream_t)s);
    }
}
