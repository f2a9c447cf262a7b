// grad_clip.hip -- global gradient norm over many tensors and clipping (include/connect6_amd.h part 7, c6_clip_*).
//
//     norm = sqrt(sum g^2),   out = g * min(1, max_norm / (norm + 1e-6))
// Two launches whatever the number of tensors: a table of chunks, made once, says where each workgroup reads and writes.  Bound by memory: every gradient in
// twice (the factor is known only after all of them) and out once.  Measured: half a billion bf16 154 + 359 us (1 GB at 6.5 TB/s, then 2 GB at 5.6: a copy
// of that size moves 5.5); 10.8 million f32 in 90 tensors 8.5 + 15 us, from the caches, their 1387 chunks going two to every third workgroup and one to the
// others; 110 thousand in 26 tensors 3.1 + 5.2 us.
#include "c6_ops.h"

#include <algorithm>
#include <vector>

namespace {

struct Chunk {                    // a piece of one tensor, the work of one workgroup at a time
    const void *src;
    void *dst;
    uint32_t n, type;
};
// 8192 elements: 32 KB or 16 KB, all of a lane's loads (8 or 4 of 16 bytes) in flight at once
constexpr uint32_t CHUNK = 8192;
// partial sums = workgroups: 4 a CU (half a billion bf16, norm + scaling: 768 147 + 377 us, 1024 155 + 353, 1280 160 + 342, 2048 160 + 413)
constexpr int MAXPART = 1024;

// over the workgroup's 256 threads, in a fixed order, the same in all of them
__device__ double block_sum(double v, double *red) {
    v = c6_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// Squares are taken and summed in 64 bits: 1e30^2 does not overflow and 1e-30^2 does not vanish.  (A conversion and a fused multiply-add an element: a
// third of what the vector unit could do while the memory delivers.)
template <typename T>
__device__ __forceinline__ double chunk_squares(const T *x, uint32_t n) {
    typedef C6Vec<T> V;
    constexpr int U = CHUNK / (256 * V::N);
    c6_u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t c = (u * 256 + threadIdx.x) * V::N;
        raw[u] = c6_u32x4{0, 0, 0, 0};
        if (c + V::N <= n) raw[u] = V::load(x + c);
    }
    double s = 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t c = (u * 256 + threadIdx.x) * V::N;
        float g[V::N];
        if (c < n && c + V::N > n) V::get_some(x + c, n - c, 0.f, g);
        else V::get(raw[u], g);
#pragma unroll
        for (int i = 0; i < V::N; i++) s = __builtin_fma((double)g[i], (double)g[i], s);
    }
    return s;
}

__global__ __launch_bounds__(256) void c6_clip_norm_kernel(const Chunk *table, int chunks, double *partial) {
    __shared__ double red[4];
    double s = 0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const Chunk k = table[c];
        C6_BY_TYPE(k.type, T, s += chunk_squares((const T *)k.src, k.n));
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ double total_norm(const double *partial, int parts, double *red) {
    double s = 0;
    for (int i = threadIdx.x; i < parts; i += 256) s += partial[i];
    return sqrt(block_sum(s, red));
}

__global__ __launch_bounds__(256) void c6_clip_finish_kernel(const double *partial, int parts, float *norm) {
    __shared__ double red[4];
    const double n = total_norm(partial, parts, red);
    if (threadIdx.x == 0) *norm = (float)n;
}

template <typename T, typename F>
__device__ __forceinline__ void chunk_scale(const T *x, T *y, uint32_t n, F f) {
    typedef C6Vec<T> V;
    constexpr int U = CHUNK / (256 * V::N);
    c6_u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t c = (u * 256 + threadIdx.x) * V::N;
        if (c + V::N <= n) raw[u] = V::load(x + c);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t c = (u * 256 + threadIdx.x) * V::N;
        if (c >= n) continue;
        const bool whole = c + V::N <= n;
        float g[V::N];
        if (whole) V::get(raw[u], g);
        else V::get_some(x + c, n - c, 0.f, g);
#pragma unroll
        for (int i = 0; i < V::N; i++) g[i] = (float)(g[i] * f);
        if (whole) V::store_past(y + c, V::put(g));
        else V::put_some(y + c, n - c, g);
    }
}

// Every workgroup adds up the partial sums itself (at most 8 KB, from the L2) instead of waiting for a launch between.  A workgroup's chunks are those of
// its namesake in the norm's pass -- the same XCD, whose L2 may still hold them -- and go from the last to the first: what was read last is still in the
// caches.  (43 MB f32: 13.3 us, from the first on 18.4; outputs written past the caches leave the next norm's pass 155 instead of 187 us of 1 GB.)
__global__ __launch_bounds__(256) void c6_clip_apply_kernel(const Chunk *table, int chunks, const double *partial, int parts, float max_norm, float *norm) {
    __shared__ double red[4];
    const double n = total_norm(partial, parts, red);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double q = (double)max_norm / (n + 1e-6);
    const float f = q > 1.0 ? 1.f : (float)q;       // a NaN norm makes f NaN
    const bool far = q < 0x1p-126;                  // f has lost bits or is 0 where a gradient times q is neither: multiplied in 64 bits
    for (int c = (int)blockIdx.x + (chunks - 1 - (int)blockIdx.x) / (int)gridDim.x * (int)gridDim.x; c >= 0; c -= gridDim.x) {
        const Chunk k = table[c];
        if (f == 1.f && k.src == k.dst) continue;   // g * 1 is g
        if (far) C6_BY_TYPE(k.type, T, chunk_scale((const T *)k.src, (T *)k.dst, k.n, q));
        else C6_BY_TYPE(k.type, T, chunk_scale((const T *)k.src, (T *)k.dst, k.n, f));
    }
}

int bad(const char *msg) { return c6_set_error(C6_ERR_BAD_ARG, msg); }

}   // namespace

struct c6_clip {
    int device = 0, chunks = 0, parts = 0;
    Chunk *table = nullptr;
};

// Memory is allocated, filled and freed beside a stream that another thread is capturing into a graph: in a thread's default mode the runtime would refuse
// these calls and end that capture.
struct AnyCapture {
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    AnyCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
    ~AnyCapture() { (void)hipThreadExchangeStreamCaptureMode(&mode); }
};
// on the thread's own stream: the default one would wait for, or be refused beside, blocking streams
static bool upload(void *to, const void *from, size_t bytes) {
    return hipMemcpyAsync(to, from, bytes, hipMemcpyHostToDevice, hipStreamPerThread) == hipSuccess && hipStreamSynchronize(hipStreamPerThread) == hipSuccess;
}

static int clip_create(int count, const void *const *grads, void *const *outs, const size_t *sizes, const int *types, int device, c6_clip **out) {
    struct Span { uintptr_t a, b; bool written; };
    std::vector<Chunk> table;
    std::vector<Span> spans;
    for (int i = 0; i < count; i++) {
        if (!c6_type_ok(types[i])) return bad("c6_clip_create: types must be C6_TYPE_F32, C6_TYPE_F16 or C6_TYPE_BF16");
        if (!sizes[i]) continue;
        const size_t es = c6_type_bytes(types[i]);
        const char *src = (const char *)grads[i];
        char *dst = outs ? (char *)outs[i] : (char *)grads[i];
        if (!src || !dst) return bad("c6_clip_create: a tensor is NULL");
        if (!c6_aligned(src, es) || !c6_aligned(dst, es)) return bad("c6_clip_create: a tensor is not aligned to its type");
        if (sizes[i] > ((size_t)1 << 46)) return bad("c6_clip_create: a tensor exceeds the address space");
        const size_t bytes = sizes[i] * es;
        if (src != dst) spans.push_back(Span{(uintptr_t)src, (uintptr_t)src + bytes, false});
        spans.push_back(Span{(uintptr_t)dst, (uintptr_t)dst + bytes, true});
        // the first chunk ends where what is written is aligned to a line of 128 bytes, and so do all the others of a long tensor
        const size_t first = CHUNK - ((uintptr_t)dst % 128) / es;
        for (size_t at = 0, n; at < sizes[i]; at += n) {
            n = std::min(at ? (size_t)CHUNK : first, sizes[i] - at);
            table.push_back(Chunk{src + at * es, dst + at * es, (uint32_t)n, (uint32_t)types[i]});
        }
    }
    if (table.size() > (size_t)1 << 30) return bad("c6_clip_create: too many elements");
    // sorted by address: an overlap shows against the furthest end so far, of anything and of what is written
    std::sort(spans.begin(), spans.end(), [](const Span &p, const Span &q) { return p.a < q.a; });
    uintptr_t end = 0, written_end = 0;
    for (const Span &s : spans) {
        if (s.a < (s.written ? end : written_end)) return bad("c6_clip_create: written memory overlaps other memory of the table");
        end = std::max(end, s.b);
        if (s.written) written_end = std::max(written_end, s.b);
    }
    if (int rc = c6_check_device(device)) return rc;
    C6DeviceScope scope(device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_clip_create: hipSetDevice");
    AnyCapture beside;
    c6_clip *c = new c6_clip();
    c->device = device;
    c->chunks = (int)table.size();
    c->parts = std::min(c->chunks, MAXPART);
    if (c->chunks && (hipMalloc(&c->table, table.size() * sizeof(Chunk)) != hipSuccess || !upload(c->table, table.data(), table.size() * sizeof(Chunk)))) {
        hipFree(c->table);
        (void)hipGetLastError();      // (reported here: not left behind for somebody else's call)
        delete c;
        return c6_set_error(C6_ERR_HIP, "c6_clip_create: no memory for the table");
    }
    *out = c;
    return C6_OK;
}

extern "C" int c6_clip_create(int count, const void *const *grads, void *const *outs, const size_t *sizes, const int *types, int device, c6_clip **out) {
    if (!out) return bad("c6_clip_create: out is NULL");
    *out = nullptr;
    if (count < 0 || (count && (!grads || !sizes || !types))) return bad("c6_clip_create: bad argument");
    try {
        return clip_create(count, grads, outs, sizes, types, device, out);
    } catch (...) {      // (the host vectors' only failure)
        return c6_set_error(C6_ERR_OVERFLOW, "c6_clip_create: out of host memory");
    }
}

extern "C" void c6_clip_destroy(c6_clip *c) {
    if (!c) return;
    C6DeviceScope scope(c->device);
    AnyCapture beside;
    hipFree(c->table);
    delete c;
}

extern "C" size_t c6_clip_workspace(const c6_clip *c) { return c ? std::max(c->parts, 1) * sizeof(double) : 0; }

static int check_call(c6_clip *c, const float *norm, bool norm_needed, const void *workspace, size_t workspace_bytes) {
    if (!c) return bad("c6_clip: NULL handle");
    if ((norm_needed && !norm) || !c6_aligned(norm, 4)) return bad("c6_clip: norm is NULL or not aligned to 4 bytes");
    if (!workspace || workspace_bytes < c6_clip_workspace(c) || !c6_aligned(workspace, 8)) return bad("c6_clip: the workspace is NULL, too small or not aligned to 8 bytes");
    return C6_OK;
}

static int enqueue(c6_clip *c, bool apply, float max_norm, float *norm, double *partial, hipStream_t s) {
    C6DeviceScope scope(c->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_clip: hipSetDevice");
    const bool ok = (!c->chunks || c6_launch(c6_clip_norm_kernel, c->parts, 256, s, c->table, c->chunks, partial)) &&
                    (apply ? c6_launch(c6_clip_apply_kernel, std::max(c->parts, 1), 256, s, c->table, c->chunks, partial, c->parts, max_norm, norm)
                           : c6_launch(c6_clip_finish_kernel, 1, 256, s, partial, c->parts, norm));
    return ok ? C6_OK : c6_set_error(C6_ERR_HIP, "c6_clip: launch failed");
}

extern "C" int c6_clip_norm(c6_clip *c, float *norm, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_call(c, norm, true, workspace, workspace_bytes)) return rc;
    return enqueue(c, false, 0.f, norm, (double *)workspace, (hipStream_t)stream);
}

extern "C" int c6_clip_apply(c6_clip *c, float max_norm, float *norm, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_call(c, norm, false, workspace, workspace_bytes)) return rc;
    if (!(max_norm >= 0.f) || max_norm > 3.402823466e38f) return bad("c6_clip_apply: max_norm must be finite and >= 0");
    return enqueue(c, true, max_norm, norm, (double *)workspace, (hipStream_t)stream);
}
