// c6_stream.h -- memory operations of the convolutions' matrix loops: weights streamed into registers some steps ahead, input slabs copied into LDS (LDS-DMA)
// one position or slice ahead, results stored between the products.
//
// Weights and results are loads and stores that the compiler sees: it keeps the registers of a load in flight, waits for them, and knows when a store has
// read its data.  (A load written in asm is done for the compiler once it is issued: where a kernel ran out of registers, one still in flight was spilled and
// its register given to something else.)  Only the LDS-DMA is asm: through the builtin every later LDS read would wait for it.  What the compiler does not
// count makes its own waits longer, never shorter.
// They are buffer operations: a scalar base and stream offset and the lane's constant 32-bit offset, no vector instruction for an address.
#pragma once
#include "c6_device.h"

__device__ __forceinline__ __amdgpu_buffer_rsrc_t c6_buffer(const void *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000);
}
// ... of memory that nothing is known about: no load from it crosses asm that may write any memory (the DMAs, waits and barriers below)
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t c6_weights(const T *w) {
    asm volatile("" : "+s"(w));
    return c6_buffer(w, -1);
}
// 16 bytes a lane at lane_off of the stream's byte soff, which passes through an empty asm: volatile statements keep their order, so the load stays behind the
// DMAs written before it
template <typename V>
__device__ __forceinline__ V c6_request(__amdgpu_buffer_rsrc_t w, unsigned lane_off, int &soff) {
    asm volatile("" : "+s"(soff));
    return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(w, lane_off, soff, 0));
}
template <typename V>
__device__ __forceinline__ void c6_put16(__amdgpu_buffer_rsrc_t z, unsigned lane_off, int soff, V v) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), z, lane_off, soff, 0);
}
// 16 bytes a lane from base + lane_off (a lane's own address) to the LDS address lds + 16 lane
__device__ __forceinline__ void c6_dma(const float *base, unsigned lane_off, int lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(lane_off), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void c6_dma(const float *from, int lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
// Vector-memory loads retire in order: with at least YOUNGER of them (c6_request) behind the last DMA and at most that many in flight, the DMA has landed.
// (Requests that the compiler adds only make the wait longer.)
template <int YOUNGER>
__device__ __forceinline__ void c6_dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(YOUNGER) : "memory"); }
// ... everybody's, and everybody's reads of LDS are done.  One statement: no LDS access gets between the wait and the barrier.
template <int YOUNGER>
__device__ __forceinline__ void c6_dma_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(YOUNGER) : "memory"); }
