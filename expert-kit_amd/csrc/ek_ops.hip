// C ABI of the operators that stand beside a layer: ek_norm (RMS norm with the residual's addition and an
// 8-bit output) and ek_linear (one int8 weight matrix on 8-bit activations).
#include "ek_host.h"
#include "ek_internal.h"

#include <algorithm>
#include <cmath>
#include <memory>
#include <mutex>

using ek::DeviceGuard;
using ek::dev_alloc;
using ek::fail;

namespace {

size_t elem_size(int dt) { return dt == EK_F32 ? 4 : dt == EK_I8 || dt == EK_F8E4M3 ? 1 : 2; }

// One device allocation that host-memory calls stage their tensors in; it grows on demand (such calls block,
// so nothing is in flight when it does).
struct Staging {
    uint8_t *ptr = nullptr;
    size_t cap = 0, used = 0;
    ek_status reserve(size_t bytes)
    {
        used = 0;
        if (bytes <= cap) return EK_OK;
        if (ptr) (void)hipFree(ptr);
        ptr = nullptr; cap = 0;
        EK_TRY(dev_alloc((void **)&ptr, bytes, "staging"));
        cap = bytes;
        return EK_OK;
    }
    static size_t part(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
    void *take(size_t bytes)
    {
        void *p = ptr + used;
        used += part(bytes);
        return p;
    }
};

ek_status check_device(int32_t dev)
{
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess) { (void)hipGetLastError(); n = 0; }
    if (dev < 0 || dev >= n) return fail(EK_HIP_ERROR, "device_id %d not available (%d HIP devices visible)", dev, n);
    return EK_OK;
}

bool misaligned(const void *p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

// Copies `bytes` from host or device memory to device memory; returns after the copy.
ek_status load_bytes(void *dst, const void *src, size_t bytes, int32_t mem)
{
    if (mem == EK_DEVICE) EK_HIP(hipDeviceSynchronize());        // the source may still be being written
    EK_HIP(hipMemcpy(dst, src, bytes, mem == EK_HOST ? hipMemcpyHostToDevice : hipMemcpyDeviceToDevice));
    EK_HIP(hipDeviceSynchronize());
    return EK_OK;
}

// Rows of one call: one workgroup of up to 1024 threads per row, and a launch holds less than 2^32 threads along a
// dimension.
constexpr int64_t kMaxRows = 65535 * 64;

}  // namespace

struct ek_norm {
    ek_norm_cfg cfg{};
    int act = 0;
    void *gain = nullptr;
    hipStream_t stream = nullptr;
    Staging staging;
    std::mutex mu;               // staging and the library's stream (blocking calls)
};

struct ek_linear {
    ek_linear_cfg cfg{};
    int act = 0;
    int64_t Kp = 0;              // in_features rounded up to whole chunks
    int32_t NT = 0;
    uint8_t *w = nullptr;        // tiles, then scales, bias
    float *bias = nullptr;
    ek::ExpertSlab *slab = nullptr;
    // rows the products cannot take as they are: 16-bit rows, rows of a length that is not whole chunks
    uint8_t *wq = nullptr;
    float *ws = nullptr;
    hipEvent_t ev = nullptr;
    bool busy = false;
    hipStream_t stream = nullptr;
    Staging staging;
    std::mutex mu;
};

namespace {

void free_norm(ek_norm *N)
{
    if (!N) return;
    (void)hipDeviceSynchronize();
    if (N->gain) (void)hipFree(N->gain);
    if (N->staging.ptr) (void)hipFree(N->staging.ptr);
    if (N->stream) (void)hipStreamDestroy(N->stream);
    delete N;
}

void free_linear(ek_linear *L)
{
    if (!L) return;
    (void)hipDeviceSynchronize();
    for (void *p : {(void *)L->w, (void *)L->slab, (void *)L->wq, (void *)L->staging.ptr})
        if (p) (void)hipFree(p);
    if (L->ev) (void)hipEventDestroy(L->ev);
    if (L->stream) (void)hipStreamDestroy(L->stream);
    delete L;
}

ek_status setup_norm(ek_norm *N, const void *gain, int32_t gain_mem)
{
    const size_t bytes = (size_t)N->cfg.hidden * 2;
    EK_TRY(dev_alloc(&N->gain, bytes, "norm gain"));
    EK_HIP(hipStreamCreateWithFlags(&N->stream, hipStreamNonBlocking));
    return load_bytes(N->gain, gain, bytes, gain_mem);
}

ek_status setup_linear(ek_linear *L, const ek_weight_desc *w, const void *bias, int32_t bias_dtype)
{
    const int64_t K = L->cfg.in_features, N = L->cfg.out_features, Kp = L->Kp, Np = (int64_t)L->NT * 16;
    const size_t tile_bytes = (size_t)Np * Kp, scale_bytes = (size_t)Np * 4;
    const size_t ses = elem_size(w->scale_dtype);
    EK_TRY(dev_alloc((void **)&L->w, tile_bytes + 2 * scale_bytes, "linear weights"));
    EK_TRY(dev_alloc((void **)&L->slab, sizeof(ek::ExpertSlab), "linear weights table"));
    const size_t rows = (size_t)L->cfg.max_rows;
    const size_t q_bytes = (rows * Kp + 255) & ~(size_t)255;
    EK_TRY(dev_alloc((void **)&L->wq, q_bytes + rows * 4, "linear workspace"));
    L->ws = (float *)(L->wq + q_bytes);
    EK_HIP(hipEventCreateWithFlags(&L->ev, hipEventDisableTiming));
    EK_HIP(hipStreamCreateWithFlags(&L->stream, hipStreamNonBlocking));
    // zero-padded copies of the matrix, its scales and the bias in the kernels' sizes
    struct Raw { uint8_t *p = nullptr; ~Raw() { if (p) (void)hipFree(p); } } raw;
    const size_t raw_scale = (size_t)Np * 4;
    EK_TRY(dev_alloc((void **)&raw.p, tile_bytes + raw_scale, "raw weights"));
    const hipMemcpyKind kind = w->mem == EK_HOST ? hipMemcpyHostToDevice : hipMemcpyDeviceToDevice;
    EK_HIP(hipDeviceSynchronize());
    EK_HIP(hipMemsetAsync(raw.p, 0, tile_bytes + raw_scale, L->stream));
    EK_HIP(hipMemcpy2DAsync(raw.p, (size_t)Kp, w->ptr, (size_t)K, (size_t)K, (size_t)N, kind, L->stream));
    EK_HIP(hipMemcpyAsync(raw.p + tile_bytes, w->scale, (size_t)N * ses, kind, L->stream));
    ek::launch_tile_weights(raw.p, EK_I8, Np, Kp, L->w, EK_I8, 0, 1, nullptr, EK_F32, L->stream);
    float *scales = (float *)(L->w + tile_bytes);
    EK_HIP(hipMemsetAsync(scales, 0, 2 * scale_bytes, L->stream));
    ek::launch_scales_to_f32(raw.p + tile_bytes, w->scale_dtype, N, scales, L->stream);
    if (bias) {
        EK_HIP(hipMemcpyAsync(raw.p + tile_bytes, bias, (size_t)N * elem_size(bias_dtype), kind, L->stream));
        L->bias = scales + Np;
        ek::launch_scales_to_f32(raw.p + tile_bytes, bias_dtype, N, L->bias, L->stream);
    }
    const ek::ExpertSlab slab{nullptr, L->w, nullptr, nullptr, scales};
    EK_HIP(hipMemcpyAsync(L->slab, &slab, sizeof slab, hipMemcpyHostToDevice, L->stream));
    EK_HIP(hipGetLastError());
    EK_HIP(hipStreamSynchronize(L->stream));
    return EK_OK;
}

// n rows of device memory -> y; the caller holds L->mu when the workspace is used.
ek_status enqueue_linear(ek_linear *L, const void *x, const float *x_scale, int64_t n, void *y, hipStream_t s)
{
    const int64_t K = L->cfg.in_features;
    ek::Q8Args a{};
    a.x = (const uint8_t *)x;
    a.x_scale = x_scale;
    if (!x_scale) {
        ek::RowQuantArgs r{};
        r.x = x; r.q = L->wq; r.scale = L->ws; r.n = n; r.H = (int32_t)K; r.q_stride = (int32_t)L->Kp;
        r.vec = K % 8 == 0 && !misaligned(x, 16);
        EK_HIP(ek::launch_row_quant(r, L->act, false, s));
        a.x = L->wq;
        a.x_scale = L->ws;
    } else if (K != L->Kp) {
        EK_HIP(ek::launch_pad_rows8(x, n, (int32_t)K, L->wq, (int32_t)L->Kp, s));
        a.x = L->wq;
    }
    a.slabs = L->slab;
    a.out = y; a.out_stride = L->cfg.out_features;
    a.N = (int32_t)L->cfg.out_features; a.NT = L->NT; a.Kdim = (int32_t)L->Kp;
    a.bias = L->bias;
    a.dense_rows = n;
    EK_HIP(ek::launch_dense_q8(a, L->act, s));
    return EK_OK;
}

}  // namespace

extern "C" {

ek_status ek_norm_create(const ek_norm_cfg *cfg, const void *gain, int32_t gain_mem, ek_norm **out)
{
    EK_GUARDED(
        if (!out) return fail(EK_INVALID_INPUT, "out is NULL");
        *out = nullptr;
        if (!cfg) return fail(EK_INVALID_INPUT, "cfg is NULL");
        if (cfg->act_dtype != EK_BF16 && cfg->act_dtype != EK_F16)
            return fail(EK_INVALID_INPUT, "act_dtype must be EK_BF16 or EK_F16 (got %d)", cfg->act_dtype);
        if (cfg->hidden < 8 || cfg->hidden % 8 || cfg->hidden > (1 << 24))
            return fail(EK_INVALID_INPUT, "hidden (%lld) must be a positive multiple of 8, at most 2^24", (long long)cfg->hidden);
        if (!(cfg->eps > 0.f) || !std::isfinite(cfg->eps))
            return fail(EK_INVALID_INPUT, "eps must be positive and finite (got %g)", (double)cfg->eps);
        if (cfg->flags) return fail(EK_INVALID_INPUT, "unknown flags 0x%x", cfg->flags);
        if (!gain) return fail(EK_WEIGHT_NOT_FOUND, "norm gain is missing");
        if (gain_mem != EK_HOST && gain_mem != EK_DEVICE) return fail(EK_INVALID_INPUT, "bad mem %d", gain_mem);
        EK_TRY(check_device(cfg->device_id));
        DeviceGuard dg(cfg->device_id);
        if (!dg.ok) return fail(EK_HIP_ERROR, "hipSetDevice(%d) failed", cfg->device_id);
        std::unique_ptr<ek_norm, void (*)(ek_norm *)> N(new ek_norm(), free_norm);
        N->cfg = *cfg;
        N->act = cfg->act_dtype == EK_BF16 ? 0 : 1;
        EK_TRY(setup_norm(N.get(), gain, gain_mem));
        *out = N.release();
        return EK_OK;
    )
}

ek_status ek_norm_forward(ek_norm *norm, const void *x, const void *residual, int64_t n, void *sum, void *y, void *q,
                          float *scale, int32_t mem, void *stream)
{
    EK_GUARDED(
        if (!norm) return fail(EK_INVALID_INPUT, "norm is NULL");
        if (n < 0 || n > kMaxRows) return fail(EK_INVALID_INPUT, "n = %lld outside [0, %lld]", (long long)n, (long long)kMaxRows);
        if (mem != EK_HOST && mem != EK_DEVICE) return fail(EK_INVALID_INPUT, "bad mem %d", mem);
        if (mem == EK_HOST && stream)
            return fail(EK_INVALID_INPUT, "host-memory calls are blocking: stream must be NULL");
        if (n > 0 && !x) return fail(EK_INVALID_INPUT, "NULL tensor pointer");
        if (n > 0 && !sum && !y && !q) return fail(EK_INVALID_INPUT, "no output asked for");
        if (sum && !residual) return fail(EK_INVALID_INPUT, "sum is x + residual: residual is NULL");
        if ((q != nullptr) != (scale != nullptr)) return fail(EK_INVALID_INPUT, "q and scale come together");
        if (sum && sum == y) return fail(EK_INVALID_INPUT, "sum and y are the same buffer");
        const size_t H = (size_t)norm->cfg.hidden;
        ek::RowQuantArgs a{};
        a.gain = norm->gain;
        a.n = n; a.H = (int32_t)H; a.q_stride = (int32_t)H; a.eps = norm->cfg.eps; a.inv_h = 1.0 / (double)H; a.vec = true;
        DeviceGuard dg(norm->cfg.device_id);
        if (!dg.ok) return fail(EK_HIP_ERROR, "hipSetDevice(%d) failed", norm->cfg.device_id);
        if (mem == EK_DEVICE) {
            if (misaligned(x, 16) || misaligned(residual, 16) || misaligned(sum, 16) || misaligned(y, 16) || misaligned(q, 8) ||
                misaligned(scale, 4))
                return fail(EK_INVALID_INPUT, "device tensors must be 16-byte aligned (q: 8, scale: 4)");
            a.x = x; a.residual = residual; a.sum = sum; a.y = y; a.q = (uint8_t *)q; a.scale = scale;
            if (stream) {
                EK_HIP(ek::launch_row_quant(a, norm->act, true, (hipStream_t)stream));
                return EK_OK;
            }
            std::lock_guard<std::mutex> lk(norm->mu);
            EK_HIP(hipDeviceSynchronize());            // a blocking call sees everything submitted before it
            EK_HIP(ek::launch_row_quant(a, norm->act, true, norm->stream));
            EK_HIP(hipStreamSynchronize(norm->stream));
            return EK_OK;
        }
        if (n == 0) return EK_OK;
        std::lock_guard<std::mutex> lk(norm->mu);
        hipStream_t s = norm->stream;
        const size_t wide = (size_t)n * H * 2;
        EK_TRY(norm->staging.reserve(4 * Staging::part(wide) + Staging::part((size_t)n * H) + Staging::part((size_t)n * 4)));
        void *dx = norm->staging.take(wide);
        EK_HIP(hipMemcpyAsync(dx, x, wide, hipMemcpyHostToDevice, s));
        a.x = dx;
        if (residual) {
            void *dr = norm->staging.take(wide);
            EK_HIP(hipMemcpyAsync(dr, residual, wide, hipMemcpyHostToDevice, s));
            a.residual = dr;
        }
        if (sum) a.sum = norm->staging.take(wide);
        if (y) a.y = norm->staging.take(wide);
        if (q) { a.q = (uint8_t *)norm->staging.take((size_t)n * H); a.scale = (float *)norm->staging.take((size_t)n * 4); }
        EK_HIP(ek::launch_row_quant(a, norm->act, true, s));
        if (sum) EK_HIP(hipMemcpyAsync(sum, a.sum, wide, hipMemcpyDeviceToHost, s));
        if (y) EK_HIP(hipMemcpyAsync(y, a.y, wide, hipMemcpyDeviceToHost, s));
        if (q) {
            EK_HIP(hipMemcpyAsync(q, a.q, (size_t)n * H, hipMemcpyDeviceToHost, s));
            EK_HIP(hipMemcpyAsync(scale, a.scale, (size_t)n * 4, hipMemcpyDeviceToHost, s));
        }
        EK_HIP(hipStreamSynchronize(s));
        return EK_OK;
    )
}

ek_status ek_norm_shape(ek_norm *norm, int64_t *hidden, int32_t *act_dtype)
{
    if (!norm || !hidden || !act_dtype) return fail(EK_INVALID_INPUT, "NULL argument");
    *hidden = norm->cfg.hidden;
    *act_dtype = norm->cfg.act_dtype;
    return EK_OK;
}

ek_status ek_norm_destroy(ek_norm *norm)
{
    EK_GUARDED(
        if (!norm) return fail(EK_INVALID_INPUT, "norm is NULL");
        DeviceGuard dg(norm->cfg.device_id);
        free_norm(norm);
        return EK_OK;
    )
}

ek_status ek_linear_create(const ek_linear_cfg *cfg, const ek_weight_desc *w, const void *bias, int32_t bias_dtype, ek_linear **out)
{
    EK_GUARDED(
        if (!out) return fail(EK_INVALID_INPUT, "out is NULL");
        *out = nullptr;
        if (!cfg) return fail(EK_INVALID_INPUT, "cfg is NULL");
        if (cfg->act_dtype != EK_BF16 && cfg->act_dtype != EK_F16)
            return fail(EK_INVALID_INPUT, "act_dtype must be EK_BF16 or EK_F16 (got %d)", cfg->act_dtype);
        // 128 * 128 * 131072 = 2^31: the longest contraction whose integer sums the kernels hold (ek_ffn_q8.hip)
        if (cfg->in_features < 1 || cfg->in_features > 131072 || cfg->out_features < 1 || cfg->out_features > (1 << 24))
            return fail(EK_INVALID_INPUT, "in_features (%lld) must be in [1, 131072] and out_features (%lld) in [1, 2^24]",
                        (long long)cfg->in_features, (long long)cfg->out_features);
        if (cfg->max_rows < 1 || cfg->max_rows > kMaxRows)
            return fail(EK_INVALID_INPUT, "max_rows (%lld) must be in [1, %lld]", (long long)cfg->max_rows, (long long)kMaxRows);
        if (cfg->flags) return fail(EK_INVALID_INPUT, "unknown flags 0x%x", cfg->flags);
        if (!w || !w->ptr) return fail(EK_WEIGHT_NOT_FOUND, "weight is missing");
        if (w->rows != cfg->out_features || w->cols != cfg->in_features)
            return fail(EK_INVALID_INPUT, "weight is [%lld,%lld], expected [%lld,%lld]", (long long)w->rows, (long long)w->cols,
                        (long long)cfg->out_features, (long long)cfg->in_features);
        if (w->mem != EK_HOST && w->mem != EK_DEVICE) return fail(EK_INVALID_INPUT, "weight: bad mem %d", w->mem);
        if (w->dtype != EK_I8) return fail(EK_INVALID_INPUT, "weight must be EK_I8 (got %d)", w->dtype);
        if (w->scale_kind != EK_SCALE_PER_CHANNEL) return fail(EK_INVALID_INPUT, "weight: int8 needs EK_SCALE_PER_CHANNEL");
        if (!w->scale) return fail(EK_WEIGHT_NOT_FOUND, "weight scale is missing");
        if (w->scale_dtype != EK_BF16 && w->scale_dtype != EK_F16 && w->scale_dtype != EK_F32)
            return fail(EK_INVALID_INPUT, "scale: bad dtype %d", w->scale_dtype);
        if (bias && bias_dtype != EK_BF16 && bias_dtype != EK_F16 && bias_dtype != EK_F32)
            return fail(EK_INVALID_INPUT, "bias: bad dtype %d", bias_dtype);
        EK_TRY(check_device(cfg->device_id));
        DeviceGuard dg(cfg->device_id);
        if (!dg.ok) return fail(EK_HIP_ERROR, "hipSetDevice(%d) failed", cfg->device_id);
        std::unique_ptr<ek_linear, void (*)(ek_linear *)> L(new ek_linear(), free_linear);
        L->cfg = *cfg;
        L->act = cfg->act_dtype == EK_BF16 ? 0 : 1;
        L->Kp = std::max<int64_t>((cfg->in_features + 63) / 64 * 64, 128);
        L->NT = (int32_t)((cfg->out_features + 15) / 16);
        EK_TRY(setup_linear(L.get(), w, bias, bias_dtype));
        *out = L.release();
        return EK_OK;
    )
}

ek_status ek_linear_forward(ek_linear *linear, const void *x, const float *x_scale, int64_t n, void *y, int32_t mem, void *stream)
{
    EK_GUARDED(
        if (!linear) return fail(EK_INVALID_INPUT, "linear is NULL");
        if (n < 0 || n > linear->cfg.max_rows)
            return fail(EK_INVALID_INPUT, "n = %lld outside [0, max_rows = %lld]", (long long)n, (long long)linear->cfg.max_rows);
        if (mem != EK_HOST && mem != EK_DEVICE) return fail(EK_INVALID_INPUT, "bad mem %d", mem);
        if (mem == EK_HOST && stream)
            return fail(EK_INVALID_INPUT, "host-memory calls are blocking: stream must be NULL");
        if (n == 0) return EK_OK;
        if (!x || !y) return fail(EK_INVALID_INPUT, "NULL tensor pointer");
        const size_t K = (size_t)linear->cfg.in_features, N = (size_t)linear->cfg.out_features;
        const bool own_rows = !x_scale || (int64_t)K != linear->Kp;     // the workspace holds the rows
        DeviceGuard dg(linear->cfg.device_id);
        if (!dg.ok) return fail(EK_HIP_ERROR, "hipSetDevice(%d) failed", linear->cfg.device_id);
        if (mem == EK_DEVICE) {
            // rows read in place go 16 bytes at a time, others by their elements; y is written in pieces that its rows' length allows
            const uintptr_t x_to = !own_rows ? 16 : x_scale ? 1 : 2, y_to = N % 8 == 0 ? 16 : N % 4 == 0 ? 8 : 2;
            if (misaligned(x, x_to) || misaligned(y, y_to) || misaligned(x_scale, 4))
                return fail(EK_INVALID_INPUT, "device tensors must be aligned: x to %d bytes, y to %d, x_scale to 4", (int)x_to, (int)y_to);
            if (stream && !own_rows) return enqueue_linear(linear, x, x_scale, n, y, (hipStream_t)stream);
            std::lock_guard<std::mutex> lk(linear->mu);
            hipStream_t s = stream ? (hipStream_t)stream : linear->stream;
            ek::WorkspaceUse use(linear->ev, &linear->busy, s);
            EK_TRY(use.begin());
            if (!stream) { EK_HIP(hipDeviceSynchronize()); use.device_idle(); }
            EK_TRY(enqueue_linear(linear, x, x_scale, n, y, s));
            if (!stream) { EK_HIP(hipStreamSynchronize(s)); use.synced(); }
            return EK_OK;
        }
        std::lock_guard<std::mutex> lk(linear->mu);
        hipStream_t s = linear->stream;
        ek::WorkspaceUse use(linear->ev, &linear->busy, s);
        EK_TRY(use.begin());
        const size_t xb = (size_t)n * K * (x_scale ? 1 : 2), yb = (size_t)n * N * 2;
        EK_TRY(linear->staging.reserve(Staging::part(xb) + Staging::part((size_t)n * 4) + Staging::part(yb)));
        void *dx = linear->staging.take(xb), *dy = linear->staging.take(yb);
        float *ds = nullptr;
        EK_HIP(hipMemcpyAsync(dx, x, xb, hipMemcpyHostToDevice, s));
        if (x_scale) {
            ds = (float *)linear->staging.take((size_t)n * 4);
            EK_HIP(hipMemcpyAsync(ds, x_scale, (size_t)n * 4, hipMemcpyHostToDevice, s));
        }
        EK_TRY(enqueue_linear(linear, dx, ds, n, dy, s));
        EK_HIP(hipMemcpyAsync(y, dy, yb, hipMemcpyDeviceToHost, s));
        EK_HIP(hipStreamSynchronize(s));
        use.synced();
        return EK_OK;
    )
}

ek_status ek_linear_shape(ek_linear *linear, int64_t *in_features, int64_t *out_features)
{
    if (!linear || !in_features || !out_features) return fail(EK_INVALID_INPUT, "NULL argument");
    *in_features = linear->cfg.in_features;
    *out_features = linear->cfg.out_features;
    return EK_OK;
}

ek_status ek_linear_destroy(ek_linear *linear)
{
    EK_GUARDED(
        if (!linear) return fail(EK_INVALID_INPUT, "linear is NULL");
        DeviceGuard dg(linear->cfg.device_id);
        free_linear(linear);
        return EK_OK;
    )
}

}  // extern "C"
