// Row kernels of the 8-bit activation path: RMS norm with the residual's addition and an int8
// output, and the quantisation of 16-bit rows.
//
// A row v is quantised symmetrically with one scale:
//   m = max|v|,  q = rint(127 v / m) (ties to even),  scale = m / 127;  a row of zeros: q = 0, scale = 0.
// For the norm, v = p * rstd with p = sum * gain and rstd = 1 / sqrt(mean(sum^2) + eps).  rstd is
// positive and the same for the whole row, so it cancels out of q: q = rint(127 p / max|p|).
// p is a product of two 16-bit values, exact in fp32 (at most 22 significant bits), so q is
// a function of the inputs alone: it does not depend on the order in which the squares are summed,
// and quant_code below gives it exactly, ties included.
//
// Bound: HBM.  A row is read once into registers by one workgroup, which reduces its sum
// of squares and its maximum together and writes everything from registers.
#include "ek_internal.h"
#include "ek_mfma.h"

namespace ek {

// rint(127 p / m) for |p| <= m.  `up` is a power of two that brings a tiny m into the range of
// normal numbers and inv = 127 / (m * up).  The fp32 product is within 2^-22 relative of the real
// value, so it decides unless it lies within 2^-15 of a half-integer; there 254 |p| is compared with the
// odd multiple of m that the half-integer stands for, both exact in fp64 (24 + 8 bits).
__device__ __forceinline__ bool quant_fast(float p, float inv, float up, float &k)
{
    const float t = (p * up) * inv;
    k = __builtin_rintf(t);
    return __builtin_fabsf(__builtin_fabsf(t - k) - 0.5f) > 0x1p-15f;   // decided
}
__device__ __forceinline__ float quant_exact(float p, float m, float inv, float up)
{
    const float a = __builtin_fabsf(p);
    const float f = __builtin_floorf((a * up) * inv);
    const double lhs = 254.0 * (double)a, rhs = (2.0 * (double)f + 1.0) * (double)m;
    const bool odd = ((int)f & 1) != 0;
    const float k = lhs > rhs || (lhs == rhs && odd) ? f + 1.f : f;
    return p < 0.f ? -k : k;
}

// 8 consecutive values of a row from index i on (i < n); vec: 16-byte loads are possible
template <typename T> __device__ __forceinline__ void load8(const T *row, int i, int n, bool vec, float *v)
{
    typedef T V8 __attribute__((ext_vector_type(8)));
    if (vec) {
        const V8 x = *(const V8 *)(row + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i + j < n ? (float)row[i + j] : 0.f;
    }
}

template <typename T> __device__ __forceinline__ void store8(T *row, int i, const float *v)
{
    typedef T V8 __attribute__((ext_vector_type(8)));
    V8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (T)v[j];
    *(V8 *)(row + i) = o;
}

// The values to quantise of 8 columns of a row: p = sum * gain (NORM; `r` receives the rounded sum), or the
// row itself.
template <typename T, bool NORM>
__device__ __forceinline__ void row_values(const RowQuantArgs &a, int64_t row, int i, float *p, float *r)
{
    load8<T>((const T *)a.x + row * a.H, i, a.H, a.vec, p);
    if constexpr (NORM) {
        if (a.residual) {
            float o[8];
            load8<T>((const T *)a.residual + row * a.H, i, a.H, true, o);
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = rnd<T>(p[j] + o[j]);
        }
        float g[8];
        load8<T>((const T *)a.gain, i, a.H, true, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) { r[j] = p[j]; p[j] = p[j] * g[j]; }
    }
}

// One workgroup per row.  NV > 0: a thread keeps its NV groups of 8 columns in registers; NV = 0:
// rows too long for that are read twice (the second time mostly from L2).
template <typename T, bool NORM, int NV, int THREADS>
__global__ __launch_bounds__(THREADS) void row_quant_kernel(RowQuantArgs a)
{
    constexpr int WAVES = THREADS / 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nvec = (a.H + 7) >> 3;
    constexpr int KEEP = NV ? NV : 1;
    float p[KEEP][8], r[NORM ? KEEP : 1][8];
    for (int64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
        // The squares are summed in fp64: no overflow for any finite input, and no dependence of the result on
        // the row's length (the kernel waits for memory: the two extra instructions per element are not seen).
        double ss = 0.0;
        float m = 0.f;
        auto take = [&](const float *pv, const float *rv) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (NORM) ss = __builtin_fma((double)rv[j], (double)rv[j], ss);
                // a NaN must not be lost: max drops it, so it is carried as an infinity
                const float v = __builtin_fabsf(pv[j]);
                m = v <= __builtin_huge_valf() ? __builtin_fmaxf(m, v) : __builtin_huge_valf();
            }
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                const int c = u * THREADS + tid;
                if (c < nvec) {
                    row_values<T, NORM>(a, row, c * 8, p[u], NORM ? r[u] : nullptr);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) { p[u][j] = 0.f; if constexpr (NORM) r[u][j] = 0.f; }
                }
            }
#pragma unroll
            for (int u = 0; u < NV; ++u) take(p[u], NORM ? r[u] : nullptr);
        } else {
            for (int c = tid; c < nvec; c += THREADS) {
                row_values<T, NORM>(a, row, c * 8, p[0], r[0]);
                take(p[0], r[0]);
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            if constexpr (NORM) ss += __shfl_xor(ss, d);
            m = __builtin_fmaxf(m, __shfl_xor(m, d));
        }
        if constexpr (WAVES > 1) {
            __shared__ double s_ss[WAVES];
            __shared__ float s_m[WAVES];
            if (lane == 0) { s_ss[wave] = ss; s_m[wave] = m; }
            __syncthreads();
            ss = s_ss[0]; m = s_m[0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) { ss += s_ss[w]; m = __builtin_fmaxf(m, s_m[w]); }
        }
        float rstd = 1.f;
        if constexpr (NORM) {
            // 1 / sqrt in fp64: the hardware's estimate and one Newton step (relative error below 2^-40)
            const double ms = ss * a.inv_h + (double)a.eps;
            const double y0 = __builtin_amdgcn_rsq(ms);
            rstd = (float)(y0 * (1.5 - 0.5 * ms * y0 * y0));      // NaN for a row with an infinity or NaN
        }
        const bool finite = m < __builtin_huge_valf();
        const float up = m < 0x1p-100f ? 0x1p64f : 1.f;
        const float inv = m > 0.f && finite ? 127.f / (m * up) : 0.f;
        if (a.scale && tid == 0) a.scale[row] = !finite ? __builtin_nanf("") : NORM ? m * rstd / 127.f : m / 127.f;

        auto give = [&](int c, const float *pv, const float *rv) {
            const int i = c * 8;
            if constexpr (NORM) {
                if (a.sum) store8<T>((T *)a.sum + row * a.H, i, rv);
                if (a.y) {
                    float o[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) o[j] = as_fp32(pv[j] * rstd);
                    store8<T>((T *)a.y + row * a.H, i, o);
                }
            }
            if (a.q) {
                float k[8];
                bool all = true;
#pragma unroll
                for (int j = 0; j < 8; ++j) all &= quant_fast(pv[j], inv, up, k[j]);
                if (!all) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float t;
                        if (!quant_fast(pv[j], inv, up, t)) k[j] = quant_exact(pv[j], m, inv, up);
                    }
                }
                uint32_t w[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j >> 2] |= ((uint32_t)(int)k[j] & 0xffu) << (8 * (j & 3));
                if (!finite) w[0] = w[1] = 0;
                *(uint2 *)(a.q + row * a.q_stride + i) = uint2{w[0], w[1]};
            }
        };
        if constexpr (NV > 0) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                const int c = u * THREADS + tid;
                if (c < nvec) give(c, p[u], NORM ? r[u] : nullptr);
            }
        } else {
            for (int c = tid; c < nvec; c += THREADS) {
                row_values<T, NORM>(a, row, c * 8, p[0], r[0]);
                give(c, p[0], r[0]);
            }
        }
        // the padding of an int8 row that the products read in whole steps
        if (a.q)
            for (int i = nvec * 8 + tid * 8; i < a.q_stride; i += THREADS * 8) *(uint2 *)(a.q + row * a.q_stride + i) = uint2{0, 0};
        if constexpr (WAVES > 1) __syncthreads();      // the next row's sums take the same LDS
    }
}

constexpr int64_t kMaxRowGroups = 1 << 21;     // a launch holds less than 2^32 threads

template <typename T, bool NORM>
static void launch_rows(const RowQuantArgs &a, hipStream_t s)
{
    const int nvec = (a.H + 7) / 8;
    const dim3 grid((unsigned)(a.n < kMaxRowGroups ? a.n : kMaxRowGroups));
#define EK_ROWS(NV, TH) hipLaunchKernelGGL((row_quant_kernel<T, NORM, NV, TH>), grid, dim3(TH), 0, s, a)
    if (nvec <= 64) EK_ROWS(1, 64);
    else if (nvec <= 256) EK_ROWS(1, 256);
    else if (nvec <= 512) EK_ROWS(2, 256);
    else if (nvec <= 1024) EK_ROWS(4, 256);
    else if (nvec <= 4096) EK_ROWS(4, 1024);
    else EK_ROWS(0, 1024);
#undef EK_ROWS
}

hipError_t launch_row_quant(const RowQuantArgs &a, int act, bool norm, hipStream_t s)
{
    if (a.n <= 0) return hipSuccess;
    if (act == 0) norm ? launch_rows<__bf16, true>(a, s) : launch_rows<__bf16, false>(a, s);
    else norm ? launch_rows<_Float16, true>(a, s) : launch_rows<_Float16, false>(a, s);
    return hipGetLastError();
}

// int8 rows of `len` bytes, back to back, into rows of `stride` bytes (a multiple of 64) whose tail is zero
__global__ __launch_bounds__(256) void pad_rows8_kernel(const uint8_t *src, int32_t len, uint8_t *dst, int32_t stride)
{
    const uint8_t *row = src + (int64_t)blockIdx.x * len;
    uint8_t *out = dst + (int64_t)blockIdx.x * stride;
    for (int col = threadIdx.x * 4; col < stride; col += 256 * 4) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < len) w |= (uint32_t)row[col + j] << (8 * j);
        *(uint32_t *)(out + col) = w;
    }
}

hipError_t launch_pad_rows8(const void *src, int64_t n, int32_t len, void *dst, int32_t stride, hipStream_t s)
{
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(pad_rows8_kernel, dim3((unsigned)n), dim3(256), 0, s, (const uint8_t *)src, len, (uint8_t *)dst, stride);
    return hipGetLastError();
}

}  // namespace ek
