// policy_ops.hip -- what a policy's logits go through before a move is chosen, and the loss they are trained on
// (include/connect6_amd.h part 7): penalties / biases / masks, cross entropy over the legal entries, and its gradient.
#include "c6_ops.h"

#include <algorithm>

namespace {

struct Rows {                     // the device's view of a c6_logits
    const void *x;
    const uint8_t *mask;
    int64_t x_stride, mask_row, mask_byte;
    int rows, width;
};

__device__ __forceinline__ bool legal(const Rows &l, int64_t r, int v) {
    return !l.mask || (l.mask[r * l.mask_row + (int64_t)(v >> 3) * l.mask_byte] >> (v & 7) & 1);
}

// the legal bits of the N entries from column c (a multiple of N) on
template <int N>
__device__ __forceinline__ uint32_t legal_bits(const Rows &l, const uint8_t *mask_row, int c) {
    return (uint32_t)mask_row[(int64_t)(c >> 3) * l.mask_byte] >> (N == 4 ? c & 4 : 0);
}

// ---- penalties, biases, masks -------------------------------------------------------------------------------------------
// A row is cut into chunks; LANES threads take one chunk: a wave for rows of up to 1024 entries (four rows a workgroup), else a workgroup per 8192.
// The chunk's logits are requested first, 16 bytes a lane and all in flight, and wait in registers while the row's history is counted in LDS:
// each chunk reads the whole history and counts the ids that fall into it (integer adds: the order does not matter).
struct Repeats {
    const int32_t *history, *len;
    const float *penalties;
    int64_t history_stride, penalties_stride;
    int cap;
};
constexpr int PROCESS_WAVE = 1024, PROCESS_BLOCK = 4096;

template <typename T, int LANES, bool HIST, bool BIAS>
__global__ __launch_bounds__(256) void c6_logits_process_kernel(Rows l, Repeats h, const float *bias, int64_t bias_stride, T *out, int64_t out_stride) {
    typedef C6Vec<T> V;
    constexpr int CHUNK = LANES == 64 ? PROCESS_WAVE : PROCESS_BLOCK, U = CHUNK / (LANES * V::N), PER = 256 / LANES;
    __shared__ uint32_t counters[HIST ? PER * CHUNK : 1];
    const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
    uint32_t *count = counters + (HIST ? part * CHUNK : 0);
    const auto meet = [] {      // one wave's LDS operations are performed in order: only the compiler has to keep them so
        if (LANES == 64) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
    };
    const int chunks = (l.width + CHUNK - 1) / CHUNK;
    const int64_t items = (int64_t)l.rows * chunks;
    for (int64_t item = (int64_t)blockIdx.x * PER + part; item < items; item += (int64_t)gridDim.x * PER) {
        const int64_t r = item / chunks;
        const int v0 = (int)(item % chunks) * CHUNK, nv = min(CHUNK, l.width - v0);
        const T *x = (const T *)l.x + r * l.x_stride + v0;
        T *o = out + r * out_stride + v0;
        const uint8_t *mask = l.mask ? l.mask + r * l.mask_row : nullptr;
        const float *b = BIAS ? bias + r * bias_stride + v0 : nullptr;
        c6_u32x4 raw[U], add[BIAS ? U : 1][V::N / 4];
        uint32_t ok[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            ok[u] = ~0u;
            if (c + V::N <= nv) raw[u] = V::load(x + c);
            if (mask && c < nv) ok[u] = legal_bits<V::N>(l, mask, v0 + c);
            if constexpr (BIAS)
                if (c + V::N <= nv)
#pragma unroll
                    for (int i = 0; i < V::N / 4; i++) add[u][i] = C6Vec<float>::load(b + c + 4 * i);
        }
        float rep = 1.f, freq = 0.f, pres = 0.f;
        if (HIST) {
            const float *p = h.penalties + r * h.penalties_stride;
            rep = p[0]; freq = p[1]; pres = p[2];
            for (int c = lane * 4; c < nv; c += LANES * 4) *reinterpret_cast<uint4 *>(count + c) = uint4{0, 0, 0, 0};
            meet();
            const int32_t *ids = h.history + r * h.history_stride;
            const int n = min(h.len ? h.len[r] : h.cap, h.cap);
            const auto seen = [&](int32_t id) {
                const uint32_t at = (uint32_t)id - (uint32_t)v0;      // (an id below v0, or below 0, wraps to far beyond nv)
                if (at < (uint32_t)nv) atomicAdd(&count[at], 1u);
            };
            constexpr int FLIGHT = 4;      // 16 ids of a lane in flight: the loop is bound by the latency of its loads
            int i = lane * 4;
            for (; i + 4 + (FLIGHT - 1) * LANES * 4 <= n; i += FLIGHT * LANES * 4) {
                c6_u32x4 q[FLIGHT];
#pragma unroll
                for (int k = 0; k < FLIGHT; k++) q[k] = C6Vec<float>::load((const float *)ids + i + k * LANES * 4);
#pragma unroll
                for (int k = 0; k < FLIGHT; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) seen((int32_t)q[k][j]);
            }
            for (; i < n; i += LANES * 4) {
                int32_t q[4];
#pragma unroll
                for (int j = 0; j < 4; j++) q[j] = i + j < n ? ids[i + j] : -1;
#pragma unroll
                for (int j = 0; j < 4; j++) seen(q[j]);
            }
            meet();
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            if (c >= nv) continue;
            const bool whole = c + V::N <= nv;
            float y[V::N];
            if (whole) V::get(raw[u], y);
            else V::get_some(x + c, nv - c, 0.f, y);
            if (HIST) {
                uint32_t k[V::N];
#pragma unroll
                for (int i = 0; i < V::N; i += 4) *reinterpret_cast<uint4 *>(k + i) = *reinterpret_cast<const uint4 *>(count + c + i);
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < V::N; i++) any |= k[i];
                if (any)
#pragma unroll
                    for (int i = 0; i < V::N; i++)
                        if (k[i]) y[i] = (y[i] > 0.f ? y[i] / rep : y[i] * rep) - (freq * (float)k[i] + pres);
            }
            if constexpr (BIAS) {
#pragma unroll
                for (int i = 0; i < V::N; i += 4) {
                    float q[4];
                    if (whole) C6Vec<float>::get(add[u][i / 4], q);
                    else C6Vec<float>::get_some(b + c + i, nv - c - i, 0.f, q);
#pragma unroll
                    for (int j = 0; j < 4; j++) y[i + j] += q[j];
                }
            }
#pragma unroll
            for (int i = 0; i < V::N; i++) y[i] = ok[u] >> i & 1 ? y[i] : -INFINITY;
            if (whole) V::store(o + c, V::put(y));
            else V::put_some(o + c, nv - c, y);
        }
        if (HIST) meet();      // the counters are read before the next item clears them
    }
}

// ---- cross entropy over the legal entries -------------------------------------------------------------------------------
struct Target {
    const void *p;
    int64_t stride;
    int kind;
};
__device__ __forceinline__ int target_index(const Target &t, int64_t r, int width) {      // -1: none
    if (t.kind == C6_TARGET_WEIGHTS) return -1;
    const int64_t i = t.kind == C6_TARGET_INDEX64 ? ((const int64_t *)t.p)[r] : ((const int32_t *)t.p)[r];
    return i >= 0 && i < width ? (int)i : -1;
}
__device__ __forceinline__ float target_weight(const Target &t, int64_t r, int v, int index) {
    return t.kind == C6_TARGET_WEIGHTS ? ((const float *)t.p)[r * t.stride + v] : (v == index ? 1.f : 0.f);
}

// target weights of the N entries from column c on, of nv columns; `index`: the column of an index target
template <int N, bool WEIGHTS>
__device__ __forceinline__ void get_weights(const float *weights, int c, int nv, int index, float (&q)[N]) {
    if (!WEIGHTS) {
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = c + i == index ? 1.f : 0.f;
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        float f[4];
        if (c + N <= nv) C6Vec<float>::get(C6Vec<float>::load(weights + c + i), f);
        else C6Vec<float>::get_some(weights + c + i, nv - c - i, 0.f, f);
#pragma unroll
        for (int j = 0; j < 4; j++) q[i + j] = f[j];
    }
}

template <typename F>
__device__ __forceinline__ float block_all(float v, F f, float *red) {
    v = c6_wave_all(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return f(f(red[0], red[1]), f(red[2], red[3]));
}

template <typename T>
__global__ __launch_bounds__(256) void c6_policy_loss_kernel(Rows l, Target t, float *loss, float *lse, float *total, T *grad, int64_t grad_stride, float scale) {
    __shared__ float red[4];
    const auto add = [](float a, float b) { return a + b; };
    for (int64_t r = blockIdx.x; r < l.rows; r += gridDim.x) {
        const T *x = (const T *)l.x + r * l.x_stride;
        const int index = target_index(t, r, l.width);
        float m = -INFINITY;
        for (int v = threadIdx.x; v < l.width; v += 256)
            if (legal(l, r, v)) m = fmaxf(m, c6_get(x[v]));
        m = block_all(m, [](float a, float b) { return fmaxf(a, b); }, red);
        if (m == -INFINITY) m = 0.f;
        // NaN is not seen by the maximum but is by the sum; the terms t (m - x) are all >= 0: nothing cancels
        float s = 0.f, w = 0.f, d = 0.f;
        for (int v = threadIdx.x; v < l.width; v += 256)
            if (legal(l, r, v)) {
                const float y = c6_get(x[v]), q = target_weight(t, r, v, index);
                s += expf(y - m);
                w += q;
                if (q != 0.f) d += q * (m - y);
            }
        s = block_all(s, add, red);
        w = block_all(w, add, red);
        d = block_all(d, add, red);
        const bool some = s != 0.f;
        if (threadIdx.x == 0) {
            loss[r] = some ? w * logf(s) + d : 0.f;
            lse[r] = some ? m + logf(s) : -INFINITY;
            total[r] = some ? w : 0.f;
        }
        if (grad) {
            const float inv = w / s;
            for (int v = threadIdx.x; v < l.width; v += 256) {
                float g = 0.f;
                if (some && legal(l, r, v)) g = scale * (expf(c6_get(x[v]) - m) * inv - target_weight(t, r, v, index));
                grad[r * grad_stride + v] = c6_put<T>(g);
            }
        }
    }
}

// The gradient from what the forward pass saved: elementwise, in chunks like those of c6_logits_process_kernel.
constexpr int GRAD_WAVE = 1024, GRAD_BLOCK = 4096;

template <typename T, int LANES, bool WEIGHTS>
__global__ __launch_bounds__(256) void c6_policy_loss_grad_kernel(Rows l, Target t, const float *lse, const float *total, const float *dloss, int64_t dloss_stride,
                                                                  T *grad, int64_t grad_stride) {
    typedef C6Vec<T> V;
    constexpr int CHUNK = LANES == 64 ? GRAD_WAVE : GRAD_BLOCK, U = CHUNK / (LANES * V::N), PER = 256 / LANES;
    const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
    const int chunks = (l.width + CHUNK - 1) / CHUNK;
    const int64_t items = (int64_t)l.rows * chunks;
    for (int64_t item = (int64_t)blockIdx.x * PER + part; item < items; item += (int64_t)gridDim.x * PER) {
        const int64_t r = item / chunks;
        const int v0 = (int)(item % chunks) * CHUNK, nv = min(CHUNK, l.width - v0);
        const T *x = (const T *)l.x + r * l.x_stride + v0;
        T *g = grad + r * grad_stride + v0;
        const float *weights = WEIGHTS ? (const float *)t.p + r * t.stride + v0 : nullptr;
        const uint8_t *mask = l.mask ? l.mask + r * l.mask_row : nullptr;
        c6_u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            if (c + V::N <= nv) raw[u] = V::load(x + c);
        }
        const int index = target_index(t, r, l.width) - v0;      // of this chunk; elsewhere or none: outside it
        const float z = lse[r], scale = dloss[r * dloss_stride], w = total[r];
        const bool some = z != -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            if (c >= nv) continue;
            const bool whole = c + V::N <= nv;
            float y[V::N], q[V::N];
            if (whole) V::get(raw[u], y);
            else V::get_some(x + c, nv - c, 0.f, y);
            get_weights<V::N, WEIGHTS>(weights, c, nv, index, q);
            uint32_t ok = some ? ~0u : 0u;
            if (mask) ok &= legal_bits<V::N>(l, mask, v0 + c);
#pragma unroll
            for (int i = 0; i < V::N; i++) y[i] = ok >> i & 1 ? scale * (w * expf(y[i] - z) - q[i]) : 0.f;
            if (whole) V::store(g + c, V::put(y));
            else V::put_some(g + c, nv - c, y);
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------
int bad(const char *msg) { return c6_set_error(C6_ERR_BAD_ARG, msg); }

// the last element a strided matrix touches stays addressable
bool fits(int64_t rows, int64_t stride, int64_t width, int64_t bytes) {
    int64_t last;
    return !__builtin_mul_overflow(rows > 0 ? rows - 1 : 0, stride, &last) && !__builtin_add_overflow(last, width, &last) &&
           !__builtin_mul_overflow(last, bytes, &last);
}

int check_logits(const c6_logits *l) {
    if (!l) return bad("logits: NULL argument");
    if (l->rows < 0 || l->width < 0) return bad("logits: negative size");
    if (!c6_type_ok(l->type)) return bad("logits: type must be C6_TYPE_F32, C6_TYPE_F16 or C6_TYPE_BF16");
    if (l->x_stride < 0 || l->mask_row < 0 || l->mask_byte < 0) return bad("logits: negative stride");
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    if (!fits(l->rows, l->x_stride, l->width, es)) return bad("logits: the matrix exceeds the address space");
    if (l->rows && l->width) {
        if (!l->x) return bad("logits: x is NULL");
        if (!c6_aligned(l->x, es)) return bad("logits: x is not aligned to its type");
    }
    return C6_OK;
}

// a written matrix: its rows do not overlap one another, and it is x itself or leaves x alone (rows of both may interleave in one buffer)
int check_written(const c6_logits *l, const void *out, int64_t stride, const char *null_msg) {
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    if (!l->rows || !l->width) return C6_OK;
    if (!out) return bad(null_msg);
    if (!c6_aligned(out, es)) return bad("logits: the output is not aligned to its type");
    if (stride < 0 || (l->rows > 1 && stride < l->width)) return bad("logits: rows of the output overlap");
    if (!fits(l->rows, stride, l->width, es)) return bad("logits: the output exceeds the address space");
    if (l->rows > 1 && out == l->x && stride != l->x_stride) return bad("logits: in place needs the same stride");
    if (out == l->x) return C6_OK;
    const int64_t a = (int64_t)(uintptr_t)l->x, b = (int64_t)(uintptr_t)out;
    const int64_t a1 = a + ((l->rows - 1) * l->x_stride + l->width) * es, b1 = b + ((l->rows - 1) * stride + l->width) * es;
    if (a1 <= b || b1 <= a) return C6_OK;
    if (l->rows > 1 && stride == l->x_stride) {      // interleaved: row r of the output lies between rows of x
        int64_t off = (b - a) % (stride * es);
        if (off < 0) off += stride * es;
        if (off >= l->width * es && stride * es - off >= l->width * es) return C6_OK;
    }
    return bad("logits: the output overlaps x without being x");
}

int check_target(const c6_logits *l, const void *target, int kind, int64_t stride) {
    if (kind != C6_TARGET_INDEX32 && kind != C6_TARGET_INDEX64 && kind != C6_TARGET_WEIGHTS) return bad("policy loss: unknown kind of target");
    if (!l->rows || (kind == C6_TARGET_WEIGHTS && !l->width)) return C6_OK;
    if (!target) return bad("policy loss: target is NULL");
    if (!c6_aligned(target, kind == C6_TARGET_INDEX64 ? 8 : 4)) return bad("policy loss: target is not aligned to its type");
    if (kind == C6_TARGET_WEIGHTS && (stride < 0 || !fits(l->rows, stride, l->width, 4))) return bad("policy loss: bad stride of the weights");
    return C6_OK;
}

// workgroups for all chunks of all rows, `per` chunks a workgroup (what exceeds the grid's limit is looped over)
unsigned grid_of(const c6_logits *l, int chunk, int per) {
    const int64_t items = (int64_t)l->rows * ((l->width + chunk - 1) / chunk);
    return (unsigned)std::min<int64_t>((items + per - 1) / per, 1 << 22);
}

Rows rows_of(const c6_logits *l) { return Rows{l->x, l->mask, l->x_stride, l->mask_row, l->mask_byte, l->rows, l->width}; }

int launched() { return hipGetLastError() == hipSuccess ? C6_OK : c6_set_error(C6_ERR_HIP, "logits: launch failed"); }

}   // namespace

extern "C" int c6_logits_process(const c6_logits *l, const int32_t *history, int64_t history_stride, const int32_t *history_len, int history_cap,
                                 const float *penalties, int64_t penalties_stride, const float *bias, int64_t bias_stride, void *out, int64_t out_stride,
                                 void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_written(l, out, out_stride, "c6_logits_process: out is NULL")) return rc;
    if (history) {
        if (history_cap < 0 || history_stride < 0 || penalties_stride < 0) return bad("c6_logits_process: negative size or stride of the history");
        if (!penalties) return bad("c6_logits_process: a history needs penalties");
        if (!c6_aligned(history, 4) || !c6_aligned(penalties, 4) || !c6_aligned(history_len, 4)) return bad("c6_logits_process: a history, its lengths and penalties are aligned to 4 bytes");
        if (!fits(l->rows, history_stride, history_cap, 4) || !fits(l->rows, penalties_stride, 3, 4)) return bad("c6_logits_process: the history exceeds the address space");
    }
    if (bias && (bias_stride < 0 || !c6_aligned(bias, 4) || !fits(l->rows, bias_stride, l->width, 4))) return bad("c6_logits_process: bad bias");
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows || !l->width) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_logits_process: hipSetDevice");
    const Repeats h{history, history_len, penalties, history_stride, penalties_stride, history_cap};
    const bool wave = l->width <= PROCESS_WAVE;
    const unsigned grid = grid_of(l, wave ? PROCESS_WAVE : PROCESS_BLOCK, wave ? 4 : 1);
#define C6_LAUNCH(LANES, HIST, BIAS)                                                                                                                        \
    C6_BY_TYPE(l->type, T, hipLaunchKernelGGL((c6_logits_process_kernel<T, LANES, HIST, BIAS>), dim3(grid), dim3(256), 0, (hipStream_t)stream, rows_of(l), \
                                              h, bias, bias_stride, (T *)out, out_stride))
#define C6_LAUNCH_LANES(LANES)                         \
    if (history && bias) C6_LAUNCH(LANES, true, true); \
    else if (history) C6_LAUNCH(LANES, true, false);   \
    else if (bias) C6_LAUNCH(LANES, false, true);      \
    else C6_LAUNCH(LANES, false, false)
    if (wave) { C6_LAUNCH_LANES(64); }
    else { C6_LAUNCH_LANES(256); }
#undef C6_LAUNCH_LANES
#undef C6_LAUNCH
    return launched();
}

extern "C" size_t c6_policy_loss_workspace(int rows, int width) { return 0; }

extern "C" int c6_policy_loss(const c6_logits *l, const void *target, int target_kind, int64_t target_stride, float *loss, float *lse, float *total, void *grad,
                              int64_t grad_stride, float grad_scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_target(l, target, target_kind, target_stride)) return rc;
    if (grad)
        if (int rc = check_written(l, grad, grad_stride, "")) return rc;
    if (l->rows && (!loss || !lse || !total)) return bad("c6_policy_loss: loss, lse or total is NULL");
    if (!c6_aligned(loss, 4) || !c6_aligned(lse, 4) || !c6_aligned(total, 4)) return bad("c6_policy_loss: loss, lse and total are aligned to 4 bytes");
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_policy_loss: hipSetDevice");
    const Target t{target, target_stride, target_kind};
    C6_BY_TYPE(l->type, T, hipLaunchKernelGGL((c6_policy_loss_kernel<T>), dim3((unsigned)std::min(l->rows, 1 << 20)), dim3(256), 0, (hipStream_t)stream, rows_of(l), t,
                                              loss, lse, total, (T *)grad, grad_stride, grad_scale));
    return launched();
}

extern "C" int c6_policy_loss_grad(const c6_logits *l, const void *target, int target_kind, int64_t target_stride, const float *lse, const float *total,
                                   const float *dloss, int64_t dloss_stride, void *grad, int64_t grad_stride, void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_target(l, target, target_kind, target_stride)) return rc;
    if (int rc = check_written(l, grad, grad_stride, "c6_policy_loss_grad: grad is NULL")) return rc;
    if (l->rows && (!lse || !total || !dloss)) return bad("c6_policy_loss_grad: lse, total or dloss is NULL");
    if (!c6_aligned(lse, 4) || !c6_aligned(total, 4) || !c6_aligned(dloss, 4)) return bad("c6_policy_loss_grad: lse, total and dloss are aligned to 4 bytes");
    if (dloss_stride < 0) return bad("c6_policy_loss_grad: negative stride");
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows || !l->width) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_policy_loss_grad: hipSetDevice");
    const Target t{target, target_stride, target_kind};
    const bool wave = l->width <= GRAD_WAVE;
    const unsigned grid = grid_of(l, wave ? GRAD_WAVE : GRAD_BLOCK, wave ? 4 : 1);
#define C6_LAUNCH(LANES, WEIGHTS)                                                                                                                          \
    C6_BY_TYPE(l->type, T, hipLaunchKernelGGL((c6_policy_loss_grad_kernel<T, LANES, WEIGHTS>), dim3(grid), dim3(256), 0, (hipStream_t)stream, rows_of(l), t, \
                                              lse, total, dloss, dloss_stride, (T *)grad, grad_stride))
    const bool weights = target_kind == C6_TARGET_WEIGHTS;
    if (wave && weights) C6_LAUNCH(64, true);
    else if (wave) C6_LAUNCH(64, false);
    else if (weights) C6_LAUNCH(256, true);
    else C6_LAUNCH(256, false);
#undef C6_LAUNCH
    return launched();
}
