// Row kernels of the 8-bit activation path: RMS norm with the residual's addition and an int8
// output, and the quantisation of 16-bit rows.
//
// A row v is quantised symmetrically with one scale:
//   m = max|v|,  q = rint(127 v / m) (ties to even),  scale = m / 127;  a row of zeros: q = 0, scale = 0.
// For the norm, v = p * rstd with p = sum * gain and rstd = 1 / sqrt(mean(sum^2) + eps).  rstd is
// positive and the same for the whole row, so it cancels out of q: q = rint(127 p / max|p|).
// p is a product of two 16-bit values, exact in fp32 (at most 22 significant bits) as long as it lies in fp32's range
// (bf16: a product beyond it counts as an infinity, one below 2^-126 loses bits), so q is a function of the inputs
// alone: it does not depend on the order in which the squares are summed, and quant8 (ek_quant.h) gives it exactly, ties
// included.
//
// Bound: HBM.  A row is read once into registers by one workgroup, which reduces its sum
// of squares and its maximum together and writes everything from registers: 8192 rows of 7168 with residual and all
// outputs, 529 MB, 96 us on MI355X = 5.5 TB/s (a copy of 4 GiB reaches 4.7).
#include "ek_internal.h"
#include "ek_mfma.h"
#include "ek_quant.h"

#include <algorithm>
#include <type_traits>

namespace ek {

// What a row holds and how it is read.
enum RowMode {
    kRowQuant = 0,       // the row itself, 16-byte loads
    kRowQuantOdd = 1,    // the row itself, whatever its length and alignment
    kRowNorm = 2,        // norm of x
    kRowNormAdd = 3      // norm of x + residual
};

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

// 8 columns as they come from memory.  All loads of a row are issued before anything is computed (a branch between them
// makes each wait for the one before: 183 us against 106 for 8192 rows of 7168); groups past the row's end
// re-read its last one and count as zeros.
template <typename T, int MODE> struct RawCols {
    typename Vec8<T>::type x, residual, gain;
    __device__ __forceinline__ void load(const RowQuantArgs &a, int64_t row, int c, int nvec)
    {
        typedef typename Vec8<T>::type V8;
        if constexpr (MODE == kRowQuantOdd) {
            const T *src = (const T *)a.x + row * a.H;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = src[min(c * 8 + j, a.H - 1)];
        } else {
            const int64_t at = row * (a.H >> 3) + min(c, nvec - 1);
            x = ((const V8 *)a.x)[at];
            if constexpr (MODE == kRowNormAdd) residual = ((const V8 *)a.residual)[at];
            if constexpr (MODE >= kRowNorm) gain = ((const V8 *)a.gain)[min(c, nvec - 1)];
        }
    }
    // p: the values to quantise; returns the rounded sum (norm)
    __device__ __forceinline__ typename Vec8<T>::type values(int c, int H, float *p) const
    {
        typename Vec8<T>::type r = x;
        const bool in = c * 8 < H;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (MODE == kRowNormAdd) r[j] = (T)((float)x[j] + (float)residual[j]);
            float v = (float)r[j];
            if constexpr (MODE >= kRowNorm) v = v * (float)gain[j];
            p[j] = (MODE == kRowQuantOdd ? c * 8 + j < H : in) ? v : 0.f;
        }
        if (MODE >= kRowNorm && !in) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = (T)0.f;
        }
        return r;
    }
};

// WPR waves per row, RPB rows per workgroup.  NV > 0: a thread keeps its NV groups of 8 columns in registers; NV = 0:
// rows too long for that are read twice (the second time mostly from L2).
template <typename T, int MODE, int NV, int WPR, int RPB>
__global__ __launch_bounds__(64 * WPR * RPB) void row_quant_kernel(RowQuantArgs a)
{
    static_assert(WPR == 1 || RPB == 1, "several rows per workgroup: one wave each");
    typedef typename Vec8<T>::type V8;
    constexpr bool NORM = MODE >= kRowNorm;
    constexpr int THREADS = 64 * WPR;                      // of a row
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tid = RPB > 1 ? lane : threadIdx.x;
    const int nvec = (a.H + 7) >> 3;
    constexpr int KEEP = NV ? NV : 1;
    for (int64_t row = RPB > 1 ? (int64_t)blockIdx.x * RPB + wave : blockIdx.x; row < a.n; row += (int64_t)gridDim.x * RPB) {
        float p[KEEP][8];
        V8 r[KEEP];
        // Squares are summed in fp64: no finite row overflows, and y is the definition's value as the nearest fp32 number, rounded to 16 bits.
        double ss = 0.0;
        uint32_t mb = 0;                                   // max |p| as bits: NaN orders behind infinity
        auto take = [&](const float *pv, const V8 &rv) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (NORM) {
                    const double f = (double)(float)rv[j];
                    ss = __builtin_fma(f, f, ss);
                }
                mb = max(mb, __builtin_bit_cast(uint32_t, pv[j]) & 0x7fffffffu);
            }
        };
        if constexpr (NV > 0) {
            RawCols<T, MODE> raw[NV];
#pragma unroll
            for (int u = 0; u < NV; ++u) raw[u].load(a, row, u * THREADS + tid, nvec);
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                r[u] = raw[u].values(u * THREADS + tid, a.H, p[u]);
                take(p[u], r[u]);
            }
        } else {
            for (int c = tid; c < nvec; c += THREADS) {
                RawCols<T, MODE> raw;
                raw.load(a, row, c, nvec);
                r[0] = raw.values(c, a.H, p[0]);
                take(p[0], r[0]);
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) {
            if constexpr (NORM) ss += __shfl_xor(ss, d);
            mb = max(mb, (uint32_t)__shfl_xor((int)mb, d));
        }
        if constexpr (WPR > 1) {
            __shared__ double s_ss[WPR];
            __shared__ uint32_t s_m[WPR];
            if (lane == 0) { s_ss[wave] = ss; s_m[wave] = mb; }
            __syncthreads();
            ss = s_ss[0]; mb = s_m[0];
#pragma unroll
            for (int w = 1; w < WPR; ++w) { ss += s_ss[w]; mb = max(mb, s_m[w]); }
            __syncthreads();                           // (the same LDS serves the next sums)
        }
        const float m = __builtin_bit_cast(float, mb);
        float rstd = 1.f, rlow = 0.f;
        double root = 1.0;
        if constexpr (NORM) {
            // 1 / sqrt in fp64: the hardware's estimate and one Newton step (relative error below 2^-40), as two fp32
            // values, so that a product with it rounds once
            const double ms = ss * a.inv_h + (double)a.eps;
            const double y0 = __builtin_amdgcn_rsq(ms);
            root = y0 * (1.5 - 0.5 * ms * y0 * y0);               // NaN for a row with an infinity or NaN
            rstd = (float)root;
            rlow = (float)(root - (double)rstd);
        }
        const QuantRow quant(m);
        if (a.scale && tid == 0) a.scale[row] = NORM ? quant.scale_of((double)m * root) : quant.scale();

        auto give = [&](int c, float *pv, const V8 &rv, auto big) {
            if constexpr (NORM) {
                const int64_t at = row * (a.H >> 3) + c;
                if (a.sum) ((V8 *)a.sum)[at] = rv;
                if (a.y) {
                    V8 o;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float v = decltype(big)::value ? pv[j] * 0x1p-64f : pv[j];
                        o[j] = (T)as_fp32(__builtin_fmaf(v, rstd, v * rlow));
                    }
                    ((V8 *)a.y)[at] = o;
                }
            }
            if (a.q) {
                const uint2 o = quant.codes(pv);
                *(uint2 *)(a.q + row * a.q_stride + c * 8) = o;
            }
        };
        auto give_row = [&](auto big) {
            if constexpr (NV > 0) {
#pragma unroll
                for (int u = 0; u < NV; ++u) {
                    const int c = u * THREADS + tid;
                    if (c < nvec) give(c, p[u], r[u], big);
                }
            } else {
                for (int c = tid; c < nvec; c += THREADS) {
                    RawCols<T, MODE> raw;
                    raw.load(a, row, c, nvec);
                    r[0] = raw.values(c, a.H, p[0]);
                    give(c, p[0], r[0], big);
                }
            }
        };
        if (NORM && std::is_same<T, __bf16>::value && rstd < 0x1p-100f) {
            // a row of values beyond 2^100: fp32 would not hold the root's low part, nor at the range's end the root itself
            rstd = (float)(root * 0x1p64);
            rlow = (float)(root * 0x1p64 - (double)rstd);
            give_row(std::true_type{});
        } else {
            give_row(std::false_type{});
        }
        // the padding of an int8 row that the products read in whole steps
        if (a.q)
            for (int i = nvec * 8 + tid * 8; i < a.q_stride; i += THREADS * 8) *(uint2 *)(a.q + row * a.q_stride + i) = uint2{0, 0};
    }
}

constexpr int64_t kMaxRowGroups = 1 << 21;     // a launch holds less than 2^32 threads

// Launch shapes: one wave per row (no barrier, four rows per workgroup) as long as a lane's share is at most four groups
// of columns and there are rows enough to fill the chip; else a workgroup per row, as wide as the row needs.
// (MI355X, 65536 rows of 2048: 98 us with 256 threads per row, 69 with a wave.)
template <typename T, int MODE>
static void launch_rows(const RowQuantArgs &a, hipStream_t s)
{
    const int nvec = (a.H + 7) / 8;
#define EK_ROWS(NV, WPR, RPB)                                                                                             \
    hipLaunchKernelGGL((row_quant_kernel<T, MODE, NV, WPR, RPB>),                                                          \
                       dim3((unsigned)std::min<int64_t>((a.n + RPB - 1) / RPB, kMaxRowGroups)), dim3(64 * WPR * RPB), 0, s, a)
    if constexpr (MODE == kRowQuantOdd) {
        if (nvec <= 256) EK_ROWS(1, 4, 1);
        else EK_ROWS(0, 16, 1);
    } else {
        if (nvec <= 64) EK_ROWS(1, 1, 4);
        else if (nvec <= 256 && a.n >= 2048) { if (nvec <= 128) EK_ROWS(2, 1, 4); else EK_ROWS(4, 1, 4); }
        else if (nvec <= 256) EK_ROWS(1, 4, 1);
        else if (nvec <= 512) EK_ROWS(2, 4, 1);
        else if (nvec <= 1024) { if (a.n < 512) EK_ROWS(1, 16, 1); else EK_ROWS(4, 4, 1); }
        else if (nvec <= 2048) EK_ROWS(2, 16, 1);
        else EK_ROWS(0, 16, 1);
    }
#undef EK_ROWS
}

template <typename T> static void launch_mode(const RowQuantArgs &a, bool norm, hipStream_t s)
{
    if (norm) a.residual ? launch_rows<T, kRowNormAdd>(a, s) : launch_rows<T, kRowNorm>(a, s);
    else a.vec ? launch_rows<T, kRowQuant>(a, s) : launch_rows<T, kRowQuantOdd>(a, s);
}

hipError_t launch_row_quant(const RowQuantArgs &a, int act, bool norm, hipStream_t s)
{
    if (a.n <= 0) return hipSuccess;
    if (act == 0) launch_mode<__bf16>(a, norm, s);
    else launch_mode<_Float16>(a, norm, s);
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
