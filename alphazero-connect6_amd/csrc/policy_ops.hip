// policy_ops.hip -- what a policy's logits go through before a move is chosen, and the loss they are trained on
// (include/connect6_amd.h part 7): penalties / biases / masks, cross entropy over the legal entries, and its gradient.
#include "c6_ops.h"
#include "c6_train.h"

#include <algorithm>
#include <initializer_list>

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

// the legal bits of the N entries from column c (a multiple of N) on, out of their byte of the mask: apart, so that no wait for the byte comes before the
// loads after it
template <int N>
__device__ __forceinline__ uint32_t legal_bits(uint32_t byte, int c) { return byte >> (N == 4 ? c & 4 : 0); }

// ---- penalties, biases, masks -------------------------------------------------------------------------------------------
// Bound by memory: every logit in and out once.  A row is cut into chunks; LANES threads take one chunk: of many rows of up to 384 entries 16 lanes each
// (lanes_of()), a wave for rows of up to 1024, else a workgroup per 4096 (in chunks of 8192 48 rows of 100003 bf16 with up to 2048 ids took a
// fifth longer: a larger chunk scans the history less often but leaves fewer waves).  The chunk's logits, mask and bias and the history's beginning are requested
// first, 16 bytes a lane and all in flight, and wait in registers while the row's history is counted in LDS: each chunk reads the whole history and counts
// the ids that fall into it (integer adds: the order does not matter).  Asking for the history's length only once the row had come cost 15 % of the time.
// Every lane loads U pieces whether its row has them or not: 361 f32 entries on 64 lanes are 90 pieces of the 256 that are asked for (the surplus ones are the
// last piece again, from the L1).
// Measured, kernel alone: 512 x 131072 f32 96 us without mask and history (5.6 TB/s; a copy of that size 99), 104 us with both; 48 x 100003 bf16 with 2048
// ids, mask and bias 9.1 us; 4096 x 361 f32 with 200 moves, legal masks and bias 7.4 us; one row of 361 2.0 us.
struct Repeats {
    const int32_t *history, *len;
    const float *penalties;
    int64_t history_stride, penalties_stride;
    int cap;
};
// entries of a chunk: of 16 lanes (four rows a wave), of a wave, of a workgroup
template <int LANES>
constexpr int chunk_of = LANES == 16 ? 384 : LANES == 64 ? 1024 : 4096;

template <typename T, int LANES, bool HIST, bool BIAS>
__global__ __launch_bounds__(256) void c6_logits_process_kernel(Rows l, Repeats h, const float *bias, int64_t bias_stride, T *out, int64_t out_stride) {
    typedef C6Vec<T> V;
    constexpr int CHUNK = chunk_of<LANES>, U = CHUNK / (LANES * V::N), PER = 256 / LANES;
    __shared__ alignas(16) uint32_t counters[HIST ? PER * CHUNK : 1];
    const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
    uint32_t *count = counters + (HIST ? part * CHUNK : 0);
    const auto meet = [] {      // one wave's LDS operations are performed in order: only the compiler has to keep them so
        if (LANES <= 64) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
    };
    const int chunks = (l.width + CHUNK - 1) / CHUNK;
    const int64_t items = (int64_t)l.rows * chunks;
    for (int64_t item = (int64_t)blockIdx.x * PER + part; item < items; item += (int64_t)gridDim.x * PER) {
        const int64_t r = item / chunks;
        const int v0 = (int)(item % chunks) * CHUNK, nv = min(CHUNK, l.width - v0);
        const int whole = nv / V::N, rest = nv % V::N, last = whole * V::N + lane;      // whole pieces; the entries behind them one a lane
        const T *x = (const T *)l.x + r * l.x_stride + v0;
        T *o = out + r * out_stride + v0;
        const uint8_t *mask = l.mask ? l.mask + r * l.mask_row : nullptr;
        const float *b = BIAS ? bias + r * bias_stride + v0 : nullptr;
        // the first ids of a lane are asked for with the row, whatever the history's length (the room of `cap` ids is the caller's)
        const int32_t *ids = HIST ? h.history + r * h.history_stride : nullptr;
        const float *p = HIST ? h.penalties + r * h.penalties_stride : nullptr;
        float rep = 1.f, freq = 0.f, pres = 0.f;
        int n = 0;
        c6_u32x4 early{0, 0, 0, 0};
        if (HIST) {
            n = min(h.len ? h.len[r] : h.cap, h.cap);
            rep = p[0]; freq = p[1]; pres = p[2];
            if (lane * 4 + 4 <= h.cap) early = C6Vec<float>::load((const float *)ids + lane * 4);
        }
        // every lane loads U pieces, behind the last one that again: no branch stands between the loads
        c6_u32x4 raw[U], add[BIAS ? U : 1][V::N / 4];
        uint32_t bits[U], tail_bits = 0xff;
        T tail = c6_put<T>(0.f);
        float tail_add = 0.f;
        if (whole) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = min(u * LANES + lane, whole - 1) * V::N;
                raw[u] = V::load(x + c);
                bits[u] = mask ? mask[(int64_t)((v0 + c) >> 3) * l.mask_byte] : 0xff;
                if constexpr (BIAS)
#pragma unroll
                    for (int i = 0; i < V::N / 4; i++) add[u][i] = C6Vec<float>::load(b + c + 4 * i);
            }
        }
        if (lane < rest) {
            tail = x[last];
            if (mask) tail_bits = mask[(int64_t)((v0 + last) >> 3) * l.mask_byte];
            if (BIAS) tail_add = b[last];
        }
        if (HIST) {
            for (int c = lane * 4; c < nv; c += LANES * 4) *reinterpret_cast<uint4 *>(count + c) = uint4{0, 0, 0, 0};
            meet();
            const auto seen = [&](int32_t id) {
                const uint32_t at = (uint32_t)id - (uint32_t)v0;      // (an id below v0, or below 0, wraps to far beyond nv)
                if (at < (uint32_t)nv) atomicAdd(&count[at], 1u);
            };
            // 8 ids of a lane in flight (64 rows of 131072 bf16 with up to 8191 ids: 4 in flight 13.3 us, 8 13.1, 16 14.5)
            constexpr int FLIGHT = 2;
            int i = lane * 4;
            if (i + 4 <= h.cap) {
#pragma unroll
                for (int j = 0; j < 4; j++) seen(i + j < n ? (int32_t)early[j] : -1);
                i += LANES * 4;
            }
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
        const auto less = [&](float y, uint32_t k) { return (y > 0.f ? y / rep : y * rep) - (freq * (float)k + pres); };
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            if (u * LANES + lane >= whole) continue;
            float y[V::N];
            V::get(raw[u], y);
            if (HIST) {
                uint32_t k[V::N], any = 0;
#pragma unroll
                for (int i = 0; i < V::N; i += 4) *reinterpret_cast<uint4 *>(k + i) = *reinterpret_cast<const uint4 *>(count + c + i);
#pragma unroll
                for (int i = 0; i < V::N; i++) any |= k[i];
                if (any)
#pragma unroll
                    for (int i = 0; i < V::N; i++) y[i] = k[i] ? less(y[i], k[i]) : y[i];
            }
            if constexpr (BIAS) {
#pragma unroll
                for (int i = 0; i < V::N; i += 4) {
                    float q[4];
                    C6Vec<float>::get(add[u][i / 4], q);
#pragma unroll
                    for (int j = 0; j < 4; j++) y[i + j] += q[j];
                }
            }
            c6_u32x4 done = V::put(y);
            V::keep(done, legal_bits<V::N>(bits[u], c));
            V::store(o + c, done);
        }
        if (lane < rest) {
            float y = c6_get(tail);
            if (HIST)
                if (const uint32_t k = count[last]) y = less(y, k);
            if (BIAS) y += tail_add;
            o[last] = c6_put<T>(tail_bits >> (last & 7) & 1 ? y : -INFINITY);
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
// -1: none.  Both kinds are read as 32-bit words, no branch before the load; width <= 2^30, so a low word below it is not negative
__device__ __forceinline__ int target_index(const Target &t, int64_t r, int width) {
    if (t.kind == C6_TARGET_WEIGHTS) return -1;
    const int words = t.kind == C6_TARGET_INDEX64 ? 2 : 1;
    const int32_t *p = (const int32_t *)t.p + r * words, low = p[0], high = p[words - 1];
    return (uint32_t)low < (uint32_t)width && (words == 1 || high == 0) ? low : -1;
}

// What is known of some legal entries of a row: their maximum m, s = sum exp(x - m), w = sum t, d = sum t (m - x).  All terms of s, w and d are
// >= 0: nothing cancels, whatever the size of the logits.  Nothing above -infinity: m = -infinity, s = 0.  The maximum does not see NaN, s does.
struct alignas(16) Part {
    float m, s, w, d;
};
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
// exp(a) as 2^(a log2 e): two half steps of |a| relative (1e-6 at |a| = 20, 5e-6 at 80) and the result's own, results below 2^-126 are 0; expf costs three times
// as many instructions
__device__ __forceinline__ float exp_of(float a) { return __builtin_amdgcn_exp2f(a * LOG2E); }
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

// p seen from a maximum M >= p.m
__device__ __forceinline__ Part from(const Part &p, float M) {
    Part q;
    q.m = M;
    q.s = p.s * exp_of(p.m - base_of(M));
    q.w = p.w;
    q.d = p.d + (p.w != 0.f && p.m != -INFINITY ? p.w * (M - p.m) : 0.f);      // (m = -infinity and w > 0: d is infinite already)
    return q;
}
// over the lanes of a row of 16 (WIDE = false) or of the wave, the same in all of them
template <bool WIDE>
__device__ __forceinline__ Part lanes_part(const Part &p, bool weights) {
    const auto top = [](float a, float b) { return fmaxf(a, b); };
    const auto add = [](float a, float b) { return a + b; };
    const auto all = [](float v, auto f) { return WIDE ? c6_wave_all(v, f) : c6_row_all(v, f); };
    Part q = from(p, all(p.m, top));
    q.s = all(q.s, add);
    if (weights) {
        q.w = all(q.w, add);
        q.d = all(q.d, add);
    }
    return q;
}
// over the lanes that share a row, the same in all of them; `space`: one Part a wave, not in use by an earlier call that some wave may still read
template <int LANES>
__device__ __forceinline__ Part block_part(const Part &p, bool weights, Part *space) {
    if (LANES == 16) return lanes_part<false>(p, weights);
    const Part q = lanes_part<true>(p, weights);
    if (LANES == 64) return q;
    if ((threadIdx.x & 63) == 0) space[threadIdx.x >> 6] = q;
    __syncthreads();
    static_assert(LANES / 64 <= 16, "one lane of a row of 16 for each wave");
    const int i = threadIdx.x & 15;
    return lanes_part<false>(i < LANES / 64 ? space[i] : Part{-INFINITY, 0.f, 0.f, 0.f}, weights);
}

// A row (or a chunk of one) in the registers of LANES lanes, in pieces of N entries (16 bytes): lane i holds the pieces i, i + LANES, ...; of the entries
// behind the last whole piece (a board's 81, 225 or 361 leave one) lane i holds the i-th.  What is not there, or not legal, is -infinity.
template <typename T, int LANES, int NV>
struct Held {
    typedef C6Vec<T> V;
    static constexpr int PIECES = NV;
    c6_u32x4 raw[NV];
    float tail;
    int whole, rest;       // whole pieces, entries behind them

    __device__ __forceinline__ Held(int width) : tail(-INFINITY), whole(width / V::N), rest(width % V::N) {
        float f[V::N];
#pragma unroll
        for (int i = 0; i < V::N; i++) f[i] = -INFINITY;
#pragma unroll
        for (int u = 0; u < NV; u++) raw[u] = V::put(f);
    }
    __device__ __forceinline__ bool has(int u, int lane) const { return lane < whole - u * LANES; }
    __device__ __forceinline__ int column(int u, int lane) const { return (u * LANES + lane) * V::N; }
    __device__ __forceinline__ void request(int u, const T *x, int lane) {
        if (has(u, lane)) raw[u] = V::load(x + u * LANES * V::N + lane * V::N);
    }
    __device__ __forceinline__ void request_tail(const T *x, int lane) {
        if (lane < rest) tail = c6_get(x[whole * V::N + lane]);
    }
    __device__ __forceinline__ void request(const T *x, int lane) {
#pragma unroll
        for (int u = 0; u < NV; u++) request(u, x, lane);
        request_tail(x, lane);
    }
};

// what was unpacked from u before is not kept for later: unpacking again is cheaper than two or four registers a word
__device__ __forceinline__ void unpack_again(c6_u32x4 &u) { asm volatile("" : "+v"(u)); }

// weights and mask of the row (or chunk), whose first column is a multiple of 8: of piece u, which begins at column c, and of single entries
struct Beside {
    const float *weights;
    const uint8_t *mask;
    int64_t byte;
    template <int N>
    __device__ __forceinline__ uint32_t bits(int, int c) const { return mask ? legal_bits<N>(mask[(int64_t)(c >> 3) * byte], c) : ~0u; }
    __device__ __forceinline__ bool legal(int c) const { return !mask || (mask[(int64_t)(c >> 3) * byte] >> (c & 7) & 1); }
    // weights: 0 where illegal
    template <int N>
    __device__ __forceinline__ void get(int u, int c, float (&q)[N]) const {
        const uint32_t ok = bits<N>(u, c);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            float f[4];
            C6Vec<float>::get(C6Vec<float>::load(weights + c + i), f);
#pragma unroll
            for (int j = 0; j < 4; j++) q[i + j] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f[j]) & C6Vec<float>::ones(ok, i + j));
        }
    }
    __device__ __forceinline__ float get(int c) const { return legal(c) ? weights[c] : 0.f; }
    template <typename H>
    __device__ __forceinline__ void settle(H &h, int lane) {
        if (!mask) return;
#pragma unroll
        for (int u = 0; u < H::PIECES; u++) {
            if (h.has(u, lane)) H::V::keep(h.raw[u], bits<H::V::N>(u, h.column(u, lane)));
            unpack_again(h.raw[u]);
        }
        if (lane < h.rest && !legal(h.whole * H::V::N + lane)) h.tail = -INFINITY;
    }
};
// ... requested all at once and held: a wave with a short row waits for memory once
template <typename T, int LANES, int NV, bool WEIGHTS>
struct Fetched {
    static constexpr int N = C6Vec<T>::N;
    uint32_t byte[NV], tail_byte;
    c6_u32x4 w[WEIGHTS ? NV : 1][N / 4];
    bool any;
    float tail_w;

    __device__ __forceinline__ Fetched(const Beside &at, const Held<T, LANES, NV> &h, int lane) : tail_byte(0xff), any(at.mask), tail_w(0.f) {
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const int c = h.column(u, lane);
            byte[u] = 0xff;
            if (!h.has(u, lane)) continue;
            if (any) byte[u] = at.mask[(int64_t)(c >> 3) * at.byte];
            if constexpr (WEIGHTS)
#pragma unroll
                for (int i = 0; i < N / 4; i++) w[u][i] = C6Vec<float>::load(at.weights + c + 4 * i);
        }
        if (lane < h.rest) {
            const int c = h.whole * N + lane;
            if (any) tail_byte = at.mask[(int64_t)(c >> 3) * at.byte];
            if (WEIGHTS) tail_w = at.weights[c];
        }
    }
    // the mask goes into the row and its weights, once
    __device__ __forceinline__ void settle(Held<T, LANES, NV> &h, int lane) {
        if (!any) return;
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const uint32_t ok = legal_bits<N>(byte[u], h.column(u, lane));
            C6Vec<T>::keep(h.raw[u], ok);
            if constexpr (WEIGHTS)
#pragma unroll
                for (int i = 0; i < N; i++) w[u][i / 4][i % 4] &= C6Vec<T>::ones(ok, i);
        }
        if (!(tail_byte >> ((h.whole * N + lane) & 7) & 1)) { h.tail = -INFINITY; tail_w = 0.f; }
    }
    template <int M>
    __device__ __forceinline__ void get(int u, int, float (&q)[M]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t word = w[WEIGHTS ? u : 0][i / 4][i % 4];
            q[i] = __builtin_bit_cast(float, word);
        }
    }
    __device__ __forceinline__ float get(int) const { return tail_w; }
};

template <bool WEIGHTS>
__device__ __forceinline__ Beside beside(const Rows &l, const Target &t, int64_t r, int v0) {
    return Beside{WEIGHTS ? (const float *)t.p + r * t.stride + v0 : nullptr, l.mask ? l.mask + r * l.mask_row + (int64_t)(v0 >> 3) * l.mask_byte : nullptr, l.mask_byte};
}

template <typename T, int LANES, int NV, bool WEIGHTS, typename At>
__device__ __forceinline__ Part part_of(Held<T, LANES, NV> &h, At &at, int lane) {
    typedef C6Vec<T> V;
    Part p{-INFINITY, 0.f, 0.f, 0.f};
    at.settle(h, lane);
    // some pieces' maximum, then their sums relative to the greatest so far: they need no piece that comes later, which may still be on its way
    const auto take = [&](const c6_u32x4 &u, float (&f)[V::N]) {
        V::get(u, f);
        float m = f[0];
#pragma unroll
        for (int i = 1; i < V::N; i++) m = fmaxf(m, f[i]);
        return m;
    };
    // a = x - base: -infinity against a weight of 0 is nothing
    const auto weigh = [&](float a, float q) {
        p.w += q;
        p.d = __builtin_fmaf(q, q != 0.f ? -a : 0.f, p.d);
    };
    const auto sum = [&](const float (&f)[V::N], bool there, int u, int c) {
        const float base = base_of(p.m);
        float a[V::N];
#pragma unroll
        for (int i = 0; i < V::N; i++) {
            a[i] = f[i] - base;
            p.s += exp_of(a[i]);
        }
        if (WEIGHTS && there) {
            float q[V::N];
            at.template get<V::N>(u, c, q);
#pragma unroll
            for (int i = 0; i < V::N; i++) weigh(a[i], q[i]);
        }
    };
    constexpr int GROUP = NV % (16 / V::N) == 0 ? 16 / V::N : LANES > 64 ? 2 : NV;      // 16 entries or 8, in short rows all
    static_assert(NV % GROUP == 0, "whole groups of pieces");
#pragma unroll
    for (int u = 0; u < NV; u += GROUP) {
        float f[GROUP][V::N], m = p.m;
#pragma unroll
        for (int j = 0; j < GROUP; j++) m = fmaxf(m, take(h.raw[u + j], f[j]));
        p = from(p, m);
#pragma unroll
        for (int j = 0; j < GROUP; j++) sum(f[j], h.has(u + j, lane), u + j, h.column(u + j, lane));
#pragma unroll
        for (int j = 0; j < GROUP; j++) unpack_again(h.raw[u + j]);
    }
    if (h.rest) {
        p = from(p, fmaxf(p.m, h.tail));
        const float a = h.tail - base_of(p.m);
        p.s += exp_of(a);
        if (WEIGHTS && lane < h.rest) weigh(a, at.get(h.whole * V::N + lane));
    }
    return p;
}
// what a row's Part says of it, and how its gradient goes: factor * exp(x - base) - scale * t (both 0 where there is nothing above -infinity)
struct Done {
    float loss, lse, total, factor, scale, base;
};
__device__ __forceinline__ Done done(const Part &p, float scale) {
    Done k;
    const float log_s = LN2 * __builtin_amdgcn_logf(p.s);
    const bool some = p.s != 0.f;
    k.base = base_of(p.m);
    k.loss = some ? p.w * log_s + p.d : 0.f;
    k.lse = some ? p.m + log_s : -INFINITY;
    k.total = some ? p.w : 0.f;
    k.factor = some ? scale * (p.w / p.s) : 0.f;
    k.scale = some ? scale : 0.f;
    return k;
}
template <typename T, bool WEIGHTS, typename At>
__device__ __forceinline__ void gradient(const c6_u32x4 &raw, const At &at, const Done &k, int index, int u, int c, T *g) {
    typedef C6Vec<T> V;
    float f[V::N];
    V::get(raw, f);
#pragma unroll
    for (int i = 0; i < V::N; i++) f[i] = k.factor * exp_of(f[i] - k.base);
    if (WEIGHTS) {
        float q[V::N];
        at.template get<V::N>(u, c, q);
#pragma unroll
        for (int i = 0; i < V::N; i++) f[i] = __builtin_fmaf(-k.scale, q[i], f[i]);
    }
    if (!WEIGHTS && (unsigned)(index - c) < (unsigned)V::N) {
#pragma unroll
        for (int i = 0; i < V::N; i++) f[i] -= c + i == index ? k.scale : 0.f;
    }
    V::store(g + c, V::put(f));
}
template <typename T, bool WEIGHTS, typename At>
__device__ __forceinline__ void gradient(float x, const At &at, const Done &k, int index, int c, T *g) {
    const float q = WEIGHTS ? at.get(c) : (c == index ? 1.f : 0.f);
    g[c] = c6_put<T>(k.factor * exp_of(x - k.base) - k.scale * q);
}

// One pass over rows that fit the registers of LANES lanes: read once, the gradient written once.  A lane takes the maximum of its own entries, the sums
// relative to that, and one reduction over the lanes joins them.  As a piece's gradient leaves, the same piece of the workgroup's next row is requested
// into its registers: loads and stores overlap, and the sums of a row begin as its first pieces arrive.
// Measured, loss and gradient: 2049 x 100003 bf16 187 us a launch among others (4.4 TB/s; 198 to 202 on its own; 1020 in three passes over each row).  There a workgroup has a CU to itself (up to 122 registers
// a lane, 16 waves) and the vector unit is busy for half the time, two exponentials an element of it: what is left over the 149 us of a copy is the part of
// that work which one row's loads do not cover, a row address aligned to two bytes (3 us), and the 2049th row.  2048 x 16000 f32 45 us (5.8 TB/s),
// 16384 x 361 bf16 against weights 11 us, 2048 x 225 f32 4 us.  The loss alone, 32768 x 361 bf16: 8.8 us for 24 MB, the vector unit busy for 4.6 of them, the rest
// the latency of one round of loads and of the reductions.  Against weights 16-bit rows of 1024 lanes and 8 pieces spill 3 registers (16 bytes of scratch).
template <typename T, int LANES, int NV, bool WEIGHTS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void c6_policy_loss_kernel(Rows l, Target t, float *loss, float *lse, float *total, T *grad, int64_t grad_stride, float scale) {
    typedef C6Vec<T> V;
    constexpr int PER = LANES < 256 ? 256 / LANES : 1;
    __shared__ Part space[2][LANES < 64 ? 1 : LANES / 64];
    const int64_t step = (int64_t)gridDim.x * PER;
    int64_t r = (int64_t)blockIdx.x * PER + (LANES == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : LANES == 16 ? threadIdx.x >> 4 : 0);
    Held<T, LANES, NV> h(l.width);
    if (r < l.rows) h.request((const T *)l.x + r * l.x_stride, threadIdx.x % LANES);
    for (int turn = 0; r < l.rows; r += step, turn ^= 1) {
        int lane = threadIdx.x % LANES;
        asm volatile("" : "+v"(lane));      // (what follows from it is computed in every turn, not kept in registers across them)
        const T *x = (const T *)l.x + r * l.x_stride;
        // what is beside a row is fetched with it where there are registers to hold it (2048 x 16001 f32 against weights: 84 instead of 119 us;
        // 2049 x 100003 bf16 with masks, against the move: 203 instead of 241), else as it is needed
        auto at = [&] {
            if constexpr (!WEIGHTS || LANES < 1024 || NV * V::N <= 32) return Fetched<T, LANES, NV, WEIGHTS>(beside<WEIGHTS>(l, t, r, 0), h, lane);
            else return beside<WEIGHTS>(l, t, r, 0);
        }();
        int index = -1;
        float played = 0.f;
        if (!WEIGHTS && l.width) {
            const int i = target_index(t, r, l.width), there = max(i, 0);
            const bool ok = legal(l, r, there);
            played = c6_get(x[there]);
            index = ok ? i : -1;
        }
        Part p = block_part<LANES>(part_of<T, LANES, NV, WEIGHTS>(h, at, lane), WEIGHTS, space[turn]);
        if (!WEIGHTS && index >= 0) { p.w = 1.f; p.d = p.m - played; }
        const Done k = done(p, scale);
        if (lane == 0) { loss[r] = k.loss; lse[r] = k.lse; total[r] = k.total; }
        const bool more = r + step < l.rows;
        const T *next = x + (more ? step * l.x_stride : 0);
        T *g = grad + r * grad_stride;
#pragma unroll
        for (int u = 0; u < NV; u++) {
            if (grad && h.has(u, lane)) gradient<T, WEIGHTS>(h.raw[u], at, k, index, u, h.column(u, lane), g);
            if (more) h.request(u, next, lane);
        }
        if (grad && lane < h.rest) gradient<T, WEIGHTS>(h.tail, at, k, index, h.whole * V::N + lane, g);
        if (more) h.request_tail(next, lane);
    }
}

// The same in two launches, for rows that do not fit or are too few to fill the card: every chunk's Part into the workspace, then each chunk joins its
// row's and writes its piece of the gradient.  3 x 131072 f32: 3.6 + 4.9 us; without a gradient 2048 x 100003 bf16 77 us (5.3 TB/s) and 7; with
// masks both together 101, where masks read only as they are needed made it 114.  With a gradient logits and weights are read twice (12 bytes an f32 entry
// instead of 8): 512 x 131072 f32 155 us against the move, 241 against weights (3.4 TB/s of the bytes read and written once), 2048 x 152064 bf16 352 and 792 us.
constexpr int SPLIT_NV = 4, JOIN_MOST = 1024;
template <typename T>
constexpr int split_chunk = 256 * SPLIT_NV * C6Vec<T>::N;

template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(256) void c6_policy_loss_part_kernel(Rows l, Target t, Part *parts, float *at) {
    __shared__ Part space[4];
    const int chunks = (l.width + split_chunk<T> - 1) / split_chunk<T>, lane = threadIdx.x;
    const int64_t items = (int64_t)l.rows * chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t r = item / chunks;
        const int v0 = (int)(item % chunks) * split_chunk<T>;
        const T *x = (const T *)l.x + r * l.x_stride;
        Held<T, 256, SPLIT_NV> h(min(l.width - v0, split_chunk<T>));
        h.request(x + v0, lane);
        Fetched<T, 256, SPLIT_NV, WEIGHTS> here(beside<WEIGHTS>(l, t, r, v0), h, lane);
        const Part p = block_part<256>(part_of<T, 256, SPLIT_NV, WEIGHTS>(h, here, lane), WEIGHTS, space);
        if (lane == 0) parts[item] = p;
        if (!WEIGHTS && lane == 0) {      // (the gradient may go where x is: the second launch does not read the entry again)
            const int index = target_index(t, r, l.width);
            if (index >= v0 && index - v0 < split_chunk<T>) at[r] = c6_get(x[index]);
        }
        __syncthreads();
    }
}

template <typename T, bool WEIGHTS>
__global__ __launch_bounds__(256) void c6_policy_loss_join_kernel(Rows l, Target t, const Part *parts, const float *at, float *loss, float *lse, float *total, T *grad,
                                                                  int64_t grad_stride, float scale) {
    typedef C6Vec<T> V;
    __shared__ Part space[4];
    const int chunks = (l.width + split_chunk<T> - 1) / split_chunk<T>, lane = threadIdx.x;
    const int per = grad ? min(chunks, JOIN_MOST) : 1;      // workgroups a row (without a gradient one): each joins ALL the row's Parts, then takes every per-th chunk
    const int64_t items = (int64_t)l.rows * per;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t r = item / per;
        const int first = (int)(item % per);
        const T *x = (const T *)l.x + r * l.x_stride;
        Held<T, 256, SPLIT_NV> h(min(l.width - first * split_chunk<T>, split_chunk<T>));
        if (grad) h.request(x + first * split_chunk<T>, lane);
        int index = -1;
        if (!WEIGHTS) {
            index = target_index(t, r, l.width);
            if (index >= 0 && !legal(l, r, index)) index = -1;
        }
        Part p{-INFINITY, 0.f, 0.f, 0.f};
        for (int i = lane; i < chunks; i += 256) {
            const Part o = parts[r * chunks + i];
            const float M = fmaxf(p.m, o.m);
            const Part a = from(p, M), b = from(o, M);
            p = Part{M, a.s + b.s, a.w + b.w, a.d + b.d};
        }
        p = block_part<256>(p, WEIGHTS, space);
        if (!WEIGHTS && index >= 0) { p.w = 1.f; p.d = p.m - at[r]; }
        const Done k = done(p, scale);
        if (first == 0 && lane == 0) { loss[r] = k.loss; lse[r] = k.lse; total[r] = k.total; }
        for (int chunk = first; grad && chunk < chunks; chunk += per) {
            const int v0 = chunk * split_chunk<T>;
            if (chunk != first) {
                h = Held<T, 256, SPLIT_NV>(min(l.width - v0, split_chunk<T>));
                h.request(x + v0, lane);
            }
            Fetched<T, 256, SPLIT_NV, WEIGHTS> here(beside<WEIGHTS>(l, t, r, v0), h, lane);
            T *g = grad + r * grad_stride + v0;
            const int at_index = index < 0 ? -1 : index - v0;      // (of another chunk: outside this one's columns)
            here.settle(h, lane);
#pragma unroll
            for (int u = 0; u < SPLIT_NV; u++)
                if (h.has(u, lane)) gradient<T, WEIGHTS>(h.raw[u], here, k, at_index, u, h.column(u, lane), g);
            if (lane < h.rest) gradient<T, WEIGHTS>(h.tail, here, k, at_index, h.whole * V::N + lane, g);
        }
        __syncthreads();
    }
}

// The gradient from what the forward pass saved: elementwise, in chunks like those of c6_logits_process_kernel.  Bound by memory: 777 x 32768 f16 against
// weights 34 us for 206 MB (6.1 TB/s), 32768 x 361 bf16 against the move 11 us (4.3 TB/s, the caches).
template <typename T, int LANES, bool WEIGHTS>
__global__ __launch_bounds__(256) void c6_policy_loss_grad_kernel(Rows l, Target t, const float *lse, const float *total, const float *dloss, int64_t dloss_stride,
                                                                  T *grad, int64_t grad_stride) {
    typedef C6Vec<T> V;
    constexpr int CHUNK = chunk_of<LANES>, U = CHUNK / (LANES * V::N), PER = 256 / LANES;
    const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
    const int chunks = (l.width + CHUNK - 1) / CHUNK;
    const int64_t items = (int64_t)l.rows * chunks;
    for (int64_t item = (int64_t)blockIdx.x * PER + part; item < items; item += (int64_t)gridDim.x * PER) {
        const int64_t r = item / chunks;
        const int v0 = (int)(item % chunks) * CHUNK, nv = min(CHUNK, l.width - v0);
        const int whole = nv / V::N, rest = nv % V::N, last = whole * V::N + lane;
        const T *x = (const T *)l.x + r * l.x_stride + v0;
        T *g = grad + r * grad_stride + v0;
        const Beside at = beside<WEIGHTS>(l, t, r, v0);
        // what the row has one of, asked for before its entries.  index: of this chunk; another chunk's lies outside its columns, and so does none
        const int index = WEIGHTS ? -1 : target_index(t, r, l.width) - v0;
        const float z = lse[r], scale = dloss[r * dloss_stride], sum = total[r];
        c6_u32x4 raw[U], w[WEIGHTS ? U : 1][V::N / 4];
        uint32_t bits[U], tail_bits = 0xff;
        T tail = c6_put<T>(0.f);
        float tail_w = 0.f;
        if (whole) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = min(u * LANES + lane, whole - 1) * V::N;
                raw[u] = V::load(x + c);
                bits[u] = at.mask ? at.mask[(int64_t)(c >> 3) * at.byte] : 0xff;
                if constexpr (WEIGHTS)
#pragma unroll
                    for (int i = 0; i < V::N / 4; i++) w[u][i] = C6Vec<float>::load(at.weights + c + 4 * i);
            }
        }
        if (lane < rest) {
            tail = x[last];
            if (at.mask) tail_bits = at.mask[(int64_t)(last >> 3) * at.byte];
            if (WEIGHTS) tail_w = at.weights[last];
        }
        const float factor = scale * sum;
        const bool some = z != -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = (u * LANES + lane) * V::N;
            if (u * LANES + lane >= whole) continue;
            float f[V::N];
            V::get(raw[u], f);
#pragma unroll
            for (int i = 0; i < V::N; i++) f[i] = factor * exp_of(f[i] - z);
            if constexpr (WEIGHTS) {
#pragma unroll
                for (int i = 0; i < V::N; i++) {
                    const uint32_t q = w[u][i / 4][i % 4];
                    f[i] = __builtin_fmaf(-scale, __builtin_bit_cast(float, q), f[i]);
                }
            } else if ((unsigned)(index - c) < (unsigned)V::N) {
#pragma unroll
                for (int i = 0; i < V::N; i++) f[i] -= c + i == index ? scale : 0.f;
            }
            const uint32_t ok = some ? legal_bits<V::N>(bits[u], c) : 0u;
#pragma unroll
            for (int i = 0; i < V::N; i++) f[i] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f[i]) & C6Vec<float>::ones(ok, i));      // 0 where illegal
            V::store(g + c, V::put(f));
        }
        if (lane < rest) {
            const float q = WEIGHTS ? tail_w : (last == index ? 1.f : 0.f);
            g[last] = c6_put<T>(some && tail_bits >> (last & 7) & 1 ? __builtin_fmaf(-scale, q, factor * exp_of(c6_get(tail) - z)) : 0.f);
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
    if (l->rows < 0 || l->width < 0 || l->width > 1 << 30) return bad("logits: a size is negative, or the width over 2^30");
    if (!c6_type_ok(l->type)) return bad("logits: type must be C6_TYPE_F32, C6_TYPE_F16 or C6_TYPE_BF16");
    if (l->x_stride < 0 || l->mask_row < 0 || l->mask_byte < 0) return bad("logits: negative stride");
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    if (!fits(l->rows, l->x_stride, l->width, es)) return bad("logits: the matrix exceeds the address space");
    int64_t bytes;      // of a row of the mask, from its first to its last
    if (l->mask && (__builtin_mul_overflow((int64_t)((l->width + 7) / 8), l->mask_byte, &bytes) || !fits(l->rows, l->mask_row, bytes, 1))) return bad("logits: the mask exceeds the address space");
    if (l->rows && l->width) {
        if (!l->x) return bad("logits: x is NULL");
        if (!c6_aligned(l->x, es)) return bad("logits: x is not aligned to its type");
    }
    return C6_OK;
}

// `rows` pieces of memory, `stride` elements apart, of `width` elements each (in bytes; sizes have passed fits())
struct Span {
    const void *p = nullptr;
    int64_t stride = 0, width = 0;
    Span(const void *p_, int64_t stride_, int64_t width_, int64_t bytes) {
        if (!p_) return;
        p = p_; stride = (int64_t)((uint64_t)stride_ * (uint64_t)bytes); width = width_ * bytes;      // (a single row's stride may be anything)
    }
};
// nothing of the one is part of the other: apart as a whole, or rows of both interleave in one buffer
bool apart(const Span &w, const Span &o, int64_t rows) {
    if (!w.p || !o.p || rows <= 0 || w.width <= 0 || o.width <= 0) return true;
    const int64_t a = (int64_t)(uintptr_t)w.p, b = (int64_t)(uintptr_t)o.p;
    if (a + (rows - 1) * w.stride + w.width <= b || b + (rows - 1) * o.stride + o.width <= a) return true;
    if (rows < 2 || w.stride < 1 || o.stride % w.stride) return false;
    int64_t off = (b - a) % w.stride;      // every row of the other lies here between two of the one
    if (off < 0) off += w.stride;
    return off >= w.width && w.stride - off >= o.width;
}
// what a call writes overlaps none of what it reads beside x
int check_apart(const c6_logits *l, const Span &out, std::initializer_list<Span> read) {
    const int64_t rows = l->rows, bytes = (l->width + 7) / 8;
    if (!out.p || !rows || !l->width) return C6_OK;
    bool ok = l->mask_byte == 1 ? apart(out, Span(l->mask, l->mask_row, bytes, 1), rows)
                                : apart(Span(out.p, 0, (rows - 1) * out.stride + out.width, 1), Span(l->mask, 0, (rows - 1) * l->mask_row + (bytes - 1) * l->mask_byte + 1, 1), 1);
    for (const Span &o : read) ok = ok && apart(out, o, rows);
    return ok ? C6_OK : bad("logits: the output overlaps another argument");
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
    return apart(Span(out, stride, l->width, es), Span(l->x, l->x_stride, l->width, es), l->rows) ? C6_OK : bad("logits: the output overlaps x without being x");
}

int check_target(const c6_logits *l, const void *target, int kind, int64_t stride) {
    if (kind != C6_TARGET_INDEX32 && kind != C6_TARGET_INDEX64 && kind != C6_TARGET_WEIGHTS) return bad("policy loss: unknown kind of target");
    if (!l->rows || (kind == C6_TARGET_WEIGHTS && !l->width)) return C6_OK;
    if (!target) return bad("policy loss: target is NULL");
    if (!c6_aligned(target, kind == C6_TARGET_INDEX64 ? 8 : 4)) return bad("policy loss: target is not aligned to its type");
    if (kind == C6_TARGET_WEIGHTS && (stride < 0 || !fits(l->rows, stride, l->width, 4))) return bad("policy loss: bad stride of the weights");
    return C6_OK;
}

Span target_span(const c6_logits *l, const void *target, int kind, int64_t stride) {
    return kind == C6_TARGET_WEIGHTS ? Span(target, stride, l->width, 4) : Span(target, 1, 1, kind == C6_TARGET_INDEX64 ? 8 : 4);
}

// Four rows a wave once that still leaves every SIMD one; 16 lanes count a history for longer, and take twice the rows for it.  Four rows a wave against
// one, 361 wide, us:  rows                         2048         4096         8192        32768
//   process, bias, f32                        3.5 / 3.3    4.2 / 4.6    6.8 / 7.3  16.6 / 18.3
//   process, bias, 50 ids, bf16               6.0 / 4.6    6.2 / 5.6    8.1 / 9.7  18.3 / 24.6
//   loss, index, bf16                         3.3 / 3.3    3.4 / 4.0    4.1 / 5.8   9.8 / 17.0
//   loss and gradient, weights, f32           4.4 / 3.9    5.5 / 5.7    8.6 / 8.7  26.8 / 25.9
//   gradient alone, weights, bf16             3.2 / 3.3    3.9 / 4.4    6.3 / 6.6  16.3 / 18.1
// (81 wide: 2048 rows within 0.2 us of one another, 32768 by half to two thirds faster).
constexpr int MANY = 4096, MANY_HISTORIES = 2 * MANY;

// the lanes that share a chunk of a row, and the workgroups for all chunks of all rows (what exceeds the grid's limit is looped over)
int lanes_of(const c6_logits *l, int many = MANY) { return l->rows >= many && l->width <= chunk_of<16> ? 16 : l->width <= chunk_of<64> ? 64 : 256; }
template <int LANES>
unsigned grid_of(const c6_logits *l) {
    const int64_t items = (int64_t)l->rows * ((l->width + chunk_of<LANES> - 1) / chunk_of<LANES>), per = 256 / LANES;
    return (unsigned)std::min<int64_t>((items + per - 1) / per, 1 << 22);
}

int cus() {
    static const int n = [] {
        int v = 0, d = 0;
        return hipGetDevice(&d) == hipSuccess && hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, d) == hipSuccess && v > 0 ? v : 256;
    }();
    return n;
}

Rows rows_of(const c6_logits *l) { return Rows{l->x, l->mask, l->x_stride, l->mask_row, l->mask_byte, l->rows, l->width}; }

int launched(bool ok) { return ok ? C6_OK : c6_set_error(C6_ERR_HIP, "logits: launch failed"); }

}   // namespace

extern "C" int c6_logits_process(const c6_logits *l, const int32_t *history, int64_t history_stride, const int32_t *history_len, int history_cap,
                                 const float *penalties, int64_t penalties_stride, const float *bias, int64_t bias_stride, void *out, int64_t out_stride,
                                 void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_written(l, out, out_stride, "c6_logits_process: out is NULL")) return rc;
    if (history) {
        if (history_cap < 0 || history_stride < 0 || penalties_stride < 0) return bad("c6_logits_process: negative size or stride of the history");
        if (history_cap > 1 << 30) return bad("c6_logits_process: a row of the history has at most 2^30 ids");      // (the kernel's index steps past its end)
        if (!penalties) return bad("c6_logits_process: a history needs penalties");
        if (!c6_aligned(history, 4) || !c6_aligned(penalties, 4) || !c6_aligned(history_len, 4)) return bad("c6_logits_process: a history, its lengths and penalties are aligned to 4 bytes");
        if (!fits(l->rows, history_stride, history_cap, 4) || !fits(l->rows, penalties_stride, 3, 4)) return bad("c6_logits_process: the history exceeds the address space");
    }
    if (bias && (bias_stride < 0 || !c6_aligned(bias, 4) || !fits(l->rows, bias_stride, l->width, 4))) return bad("c6_logits_process: bad bias");
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    if (int rc = check_apart(l, Span(out, out_stride, l->width, es), {Span(bias, bias_stride, l->width, 4), Span(history, history_stride, history_cap, 4),
                                                                    Span(history ? history_len : nullptr, 1, 1, 4), Span(history ? penalties : nullptr, penalties_stride, 3, 4)})) return rc;
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows || !l->width) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_logits_process: hipSetDevice");
    const Repeats h{history, history_len, penalties, history_stride, penalties_stride, history_cap};
    bool ok = false;
#define C6_LAUNCH(LANES, HIST, BIAS)                                                                                                                        \
    C6_BY_TYPE(l->type, T, ok = c6_launch(c6_logits_process_kernel<T, LANES, HIST, BIAS>, grid_of<LANES>(l), 256, (hipStream_t)stream, rows_of(l), h, bias, bias_stride, \
                                          (T *)out, out_stride))
#define C6_LAUNCH_LANES(LANES)                         \
    if (history && bias) C6_LAUNCH(LANES, true, true); \
    else if (history) C6_LAUNCH(LANES, true, false);   \
    else if (bias) C6_LAUNCH(LANES, false, true);      \
    else C6_LAUNCH(LANES, false, false)
    switch (lanes_of(l, history ? MANY_HISTORIES : MANY)) {
    case 16: C6_LAUNCH_LANES(16); break;
    case 64: C6_LAUNCH_LANES(64); break;
    default: C6_LAUNCH_LANES(256);
    }
#undef C6_LAUNCH_LANES
#undef C6_LAUNCH
    return launched(ok);
}

// Which way the loss goes, by the pieces of N entries (16 bytes) in a row.  The registers of 64, 256 or 1024 lanes hold up to 16384 (against weights, which
// need registers of their own, 8192).  Split into chunks go
//   longer rows;
//   rows of over 8192 pieces that are too few for a workgroup each to fill the card (3 x 100003 bf16: 17.7 us in one workgroup a row).  The border of 128 rows
//   is half of the CUs, not a measured one: from there to some 600 rows the last round of workgroups leaves much of the card idle (with a gradient, bf16, 80001
//   wide: 129 rows 17 us, 257 28, 300 33, 512 36);
//   without a gradient nothing need be held: from 2048 pieces on small workgroups are faster (2048 x 100003 bf16: 77 against 113 us; few rows: one launch is).
static bool splits(int64_t rows, int64_t width, int n, bool weights, bool grad) {
    const int64_t pieces = (width + n - 1) / n;
    return pieces > (weights ? 8192 : 16384) || (rows <= 128 ? pieces > 8192 : !grad && pieces > 2048);
}
static size_t split_bytes(int64_t rows, int64_t width, int n) {
    const int64_t chunk = 256 * SPLIT_NV * n;
    return (size_t)rows * ((size_t)((width + chunk - 1) / chunk) * sizeof(Part) + sizeof(float));
}

extern "C" size_t c6_policy_loss_workspace(int rows, int width) {
    size_t need = 0;
    for (int n : {4, 8})      // whatever the type
        if (rows > 0 && splits(rows, width, n, true, false)) need = std::max(need, split_bytes(rows, width, n));
    return need;
}

template <typename T, bool WEIGHTS>
static bool loss_launch(const c6_logits *l, const Target &t, float *loss, float *lse, float *total, T *grad, int64_t grad_stride, float scale, void *workspace, hipStream_t s) {
    constexpr int N = C6Vec<T>::N;
    const Rows rows = rows_of(l);
    if (splits(l->rows, l->width, N, WEIGHTS, grad != nullptr)) {
        const int64_t chunks = (l->width + split_chunk<T> - 1) / split_chunk<T>, items = l->rows * chunks;
        Part *parts = (Part *)workspace;
        float *at = (float *)(parts + items);
        const unsigned grid = (unsigned)std::min<int64_t>(items, 1 << 22), join = (unsigned)std::min<int64_t>(l->rows * (grad ? std::min<int64_t>(chunks, JOIN_MOST) : 1), 1 << 22);
        return c6_launch(c6_policy_loss_part_kernel<T, WEIGHTS>, grid, 256, s, rows, t, parts, at) &&
               c6_launch(c6_policy_loss_join_kernel<T, WEIGHTS>, join, 256, s, rows, t, parts, at, loss, lse, total, grad, grad_stride, scale);
    }
#define C6_LAUNCH(LANES, NV, RESIDENT)                                                                                                                                       \
    return c6_launch(c6_policy_loss_kernel<T, LANES, NV, WEIGHTS>, (unsigned)std::min<int64_t>(LANES < 256 ? ((int64_t)l->rows * LANES + 255) / 256 : l->rows, (int64_t)cus() * RESIDENT), \
                     LANES < 256 ? 256 : LANES, s, rows, t, loss, lse, total, grad, grad_stride, scale)
    // Pieces beyond the row take part in its sums all the same.  From 2048 on the pieces held go up by a half or a third, below by two (four short rows a wave: by a
    // half or a third): by two everywhere 300 x 80001 bf16 took 37.1 us instead of 33.3, 2048 x 20000 f32 85.7 instead of 80.3, 2048 x 24000 bf16 against weights
    // 92.0 instead of 85.5.  14 pieces of 1024 lanes: rows of 12289 to 14336 pieces, among them a 16-bit vocabulary of 100 thousand (2049 x 100003 198 -> 194.5 us).
    // (Skipped by a branch surplus pieces cost 2048 x 128000 bf16, where there are none, 8 %.)
    const int pieces = (l->width + N - 1) / N;
    const bool many = l->rows >= MANY;
    if (many && pieces <= 32) C6_LAUNCH(16, 2, 1 << 14);
    else if (many && pieces <= 48) C6_LAUNCH(16, 3, 1 << 14);
    else if (many && pieces <= 64) C6_LAUNCH(16, 4, 1 << 14);
    else if (many && pieces <= 96) C6_LAUNCH(16, 6, 1 << 14);
    else if (pieces <= 64) C6_LAUNCH(64, 1, 1 << 14);
    else if (pieces <= 128) C6_LAUNCH(64, 2, 1 << 14);
    else if (pieces <= 256) C6_LAUNCH(64, 4, 1 << 14);
    else if (pieces <= 512) C6_LAUNCH(256, 2, 1 << 14);
    else if (pieces <= 1024) C6_LAUNCH(256, 4, 1 << 14);
    else if (pieces <= 2048) C6_LAUNCH(512, 4, 1 << 14);
    else if (pieces <= 3 * 1024) C6_LAUNCH(512, 6, 1 << 14);
    else if (pieces <= 4096) C6_LAUNCH(512, 8, 1 << 14);
    else if constexpr (WEIGHTS) {
        if (pieces <= 6144) C6_LAUNCH(1024, 6, 1);
        else C6_LAUNCH(1024, 8, 1);
    }
    else if (pieces <= 6144) C6_LAUNCH(512, 12, 1 << 14);
    else if (pieces <= 8192) C6_LAUNCH(512, 16, 1 << 14);
    else if (pieces <= 12288) C6_LAUNCH(1024, 12, 1);
    else if (pieces <= 14336) C6_LAUNCH(1024, 14, 1);
    else C6_LAUNCH(1024, 16, 1);
#undef C6_LAUNCH
}

extern "C" int c6_policy_loss(const c6_logits *l, const void *target, int target_kind, int64_t target_stride, float *loss, float *lse, float *total, void *grad,
                              int64_t grad_stride, float grad_scale, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_target(l, target, target_kind, target_stride)) return rc;
    if (grad)
        if (int rc = check_written(l, grad, grad_stride, "")) return rc;
    if (l->rows && (!loss || !lse || !total)) return bad("c6_policy_loss: loss, lse or total is NULL");
    if (!c6_aligned(loss, 4) || !c6_aligned(lse, 4) || !c6_aligned(total, 4)) return bad("c6_policy_loss: loss, lse and total are aligned to 4 bytes");
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    const Span t_span = target_span(l, target, target_kind, target_stride);
    if (int rc = check_apart(l, Span(grad, grad_stride, l->width, es), {t_span, Span(loss, 1, 1, 4), Span(lse, 1, 1, 4), Span(total, 1, 1, 4)})) return rc;
    for (const float *stat : {loss, lse, total})
        if (int rc = check_apart(l, Span(stat, 1, 1, 4), {t_span, Span(l->x, l->x_stride, l->width, es)})) return rc;
    const int n = l->type == C6_TYPE_F32 ? 4 : 8;
    if (l->rows && splits(l->rows, l->width, n, target_kind == C6_TARGET_WEIGHTS, grad != nullptr) && (!workspace || workspace_bytes < split_bytes(l->rows, l->width, n) || !c6_aligned(workspace, alignof(Part))))
        return bad("c6_policy_loss: the workspace is NULL, smaller than c6_policy_loss_workspace() or not aligned to 16 bytes");
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_policy_loss: hipSetDevice");
    const Target t{target, target_stride, target_kind};
    bool ok = false;
    C6_BY_TYPE(l->type, T, const auto launch = target_kind == C6_TARGET_WEIGHTS ? loss_launch<T, true> : loss_launch<T, false>;
               ok = launch(l, t, loss, lse, total, (T *)grad, grad_stride, grad_scale, workspace, (hipStream_t)stream));
    return launched(ok);
}

extern "C" int c6_policy_loss_grad(const c6_logits *l, const void *target, int target_kind, int64_t target_stride, const float *lse, const float *total,
                                   const float *dloss, int64_t dloss_stride, void *grad, int64_t grad_stride, void *stream) {
    if (int rc = check_logits(l)) return rc;
    if (int rc = check_target(l, target, target_kind, target_stride)) return rc;
    if (int rc = check_written(l, grad, grad_stride, "c6_policy_loss_grad: grad is NULL")) return rc;
    if (l->rows && (!lse || !total || !dloss)) return bad("c6_policy_loss_grad: lse, total or dloss is NULL");
    if (!c6_aligned(lse, 4) || !c6_aligned(total, 4) || !c6_aligned(dloss, 4)) return bad("c6_policy_loss_grad: lse, total and dloss are aligned to 4 bytes");
    if (dloss_stride < 0 || !fits(l->rows, dloss_stride, 1, 4)) return bad("c6_policy_loss_grad: bad stride of dloss");
    const int64_t es = (int64_t)c6_type_bytes(l->type);
    if (int rc = check_apart(l, Span(grad, grad_stride, l->width, es), {target_span(l, target, target_kind, target_stride), Span(lse, 1, 1, 4), Span(total, 1, 1, 4), Span(dloss, dloss_stride, 1, 4)}))
        return rc;
    if (int rc = c6_check_device(l->device)) return rc;
    if (!l->rows || !l->width) return C6_OK;
    C6DeviceScope scope(l->device);
    if (!scope.ok) return c6_set_error(C6_ERR_HIP, "c6_policy_loss_grad: hipSetDevice");
    const Target t{target, target_stride, target_kind};
#define C6_LAUNCH(LANES, WEIGHTS)                                                                                                                          \
    C6_BY_TYPE(l->type, T, ok = c6_launch(c6_policy_loss_grad_kernel<T, LANES, WEIGHTS>, grid_of<LANES>(l), 256, (hipStream_t)stream, rows_of(l), t, lse, total, dloss, \
                                          dloss_stride, (T *)grad, grad_stride))
    const bool weights = target_kind == C6_TARGET_WEIGHTS;
    bool ok = false;
    switch (lanes_of(l)) {
    case 16: if (weights) C6_LAUNCH(16, true); else C6_LAUNCH(16, false); break;
    case 64: if (weights) C6_LAUNCH(64, true); else C6_LAUNCH(64, false); break;
    default: if (weights) C6_LAUNCH(256, true); else C6_LAUNCH(256, false);
    }
#undef C6_LAUNCH
    return launched(ok);
}

// The trainer's batch in the operator's terms; a wave a position.  Visits are summed and divided in 64 bits: finite ones of any size have a finite sum (with sums
// below 2^24 and whole visits the same bits as in 32: one rounding of the same quotient).
__global__ __launch_bounds__(256) void c6t_policy_targets_kernel(int B, int cells, const float *boards, const float *poses, const float *visits, uint8_t *mask, int *index,
                                                                 float *weights) {
    const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6), bytes = (cells + 7) / 8;
    if (b >= B) return;
    double sum = 0;
    for (int v0 = 0; v0 < cells; v0 += 64) {
        const int v = v0 + lane;
        const bool empty = v < cells && boards[(size_t)b * cells + v] == 0.f;
        const uint64_t bits = __ballot(empty);
        if (lane < 8 && v0 / 8 + lane < bytes) mask[(size_t)b * bytes + v0 / 8 + lane] = (uint8_t)(bits >> (8 * lane));
        if (visits && empty) sum += visits[(size_t)b * cells + v];
    }
    if (!visits) {
        if (lane == 0) index[b] = (int)poses[b];
        return;
    }
    sum = c6_wave_sum(sum);
    for (int v = lane; v < cells; v += 64) weights[(size_t)b * cells + v] = sum > 0 ? (float)(visits[(size_t)b * cells + v] / sum) : 0.f;
}
void c6t_policy_targets(int B, int cells, const float *boards, const float *poses, const float *visits, unsigned char *mask, int *index, float *weights, hipStream_t s) {
    hipLaunchKernelGGL(c6t_policy_targets_kernel, dim3((B + 3) / 4), dim3(256), 0, s, B, cells, boards, poses, visits, mask, index, weights);
}
