// grads.h — device side of the gc_grads table (include/gcodec.h): many gradient
// tensors of float32, float16 and bfloat16 addressed as one flat sequence of n
// elements.
//
// Flat element e of tensor s (start[s] <= e < start[s + 1]) lives at
// ptr[s] + (e - start[s]).  A wave takes ranges of the flat sequence, so the
// work of a launch is even whatever the tensors' sizes are, and walks the
// pieces of its range that lie in one tensor each.  The tensor, the piece and
// their addresses are the same for the 64 lanes: they stay in scalar
// registers, and the lanes of a piece read or write consecutive vectors.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gc_device.h"

namespace gc {

constexpr uint32_t kTF32 = 0, kTF16 = 1, kTBF16 = 2;  // element types in a record's top byte

struct GradRec {  // = two words of gc_grads.rec
    uint64_t pt;     // type << 56 | address
    uint64_t start;  // first flat element
};

struct GradArg {
    const GradRec *rec;  // count records and a closing one (start = n)
    uint32_t count;
};

// Tables of up to kLdsRecs tensors are copied to LDS by each block: a lookup
// is then two LDS reads instead of two dependent trips to the L2.  Decoding 246M
// bfloat16 of 38 tensors takes 252 us so and 335 without, clipping 10,000
// elements of 120 tensors 11.7 and 13.4; long passes over few tensors do not
// notice (the norm of 23.5M in 161: 18.4 and 18.2).
constexpr uint32_t kLdsRecs = 1024;

__device__ __forceinline__ uint32_t uni32(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uni64(uint64_t v)
{
    return (uint64_t)uni32((uint32_t)(v >> 32)) << 32 | uni32((uint32_t)v);
}
__device__ __forceinline__ uint32_t lane_id() { return threadIdx.x & 63u; }
__device__ __forceinline__ uint32_t wave_id() { return uni32(threadIdx.x >> 6); }

// the block's copy of a table (followed by a barrier of the caller's)
__device__ __forceinline__ void stage_table(const GradArg &g, GradRec *lds)
{
    for (uint32_t i = threadIdx.x; i <= g.count; i += blockDim.x)
        lds[i] = g.rec[i];
}

// the tensor that holds flat element e < n: the last s with start[s] <= e
// (empty tensors share their successor's start and are passed over).  The 64
// lanes probe 64 records at a time, so a table of T tensors takes
// ceil(log64 T) rounds.  Every lane of the wave must be active.
__device__ __forceinline__ uint32_t grad_find(const GradRec *rec, uint32_t count, uint64_t e)
{
    uint32_t lo = 0, len = count;  // start[lo] <= e < start[lo + len]
    while (len > 1) {
        const uint32_t step = (len + 63) >> 6;
        const uint32_t off = lane_id() * step;
        const bool le = off < len && rec[lo + off].start <= e;
        const uint32_t c = __popcll(__ballot(le)) - 1;  // lane 0 always holds
        lo += c * step;
        len = min(step, len - c * step);
    }
    return lo;
}

// f(s, type, base, start, a, b) for every piece [a, b) of the non-empty flat
// range [lo, hi), hi <= n, whose first element is in tensor s; s the piece's
// tensor, base its address, start its first element
template <class F>
__device__ __forceinline__ void grad_walk(const GradRec *rec, uint32_t s, uint64_t lo, uint64_t hi, F f)
{
    uint64_t a = lo;
    for (;;) {
        const uint64_t pt = uni64(rec[s].pt), start = uni64(rec[s].start), end = uni64(rec[s + 1].start);
        const uint64_t b = end < hi ? end : hi;
        if (b > a)
            f(s, (uint32_t)(pt >> 56), pt & 0x00ffffffffffffffull, start, a, b);
        if (end >= hi)  // start[count] = n >= hi: s never passes the last tensor
            return;
        a = end;
        ++s;
    }
}

// Whether [lo, hi), which begins in tensor s, spans more than `many` tensors
// (empty ones count).  A walk waits for the memory once a piece: a range of many
// takes its elements lane by lane instead, each lane with the tensors of its own
// (grad_lane).
__device__ __forceinline__ bool grad_many(const GradRec *rec, uint32_t count, uint32_t s, uint64_t hi, uint32_t many)
{
    return uni64(rec[min(s + many, count)].start) < hi;
}

// the lane's tensor of element e, known to be in s .. last
__device__ __forceinline__ uint32_t grad_lane(const GradRec *rec, uint32_t s, uint32_t last, uint64_t e)
{
    while (s < last) {
        const uint32_t mid = (s + last + 1) >> 1;
        if (rec[mid].start <= e)
            s = mid;
        else
            last = mid - 1;
    }
    return s;
}

// ---------------------------------------------------------------------------
// vectors of V elements at any element-aligned address.  Global memory takes
// 16-byte accesses at element alignment on gfx950; a misaligned one costs at
// most one more cache line for a whole wave's access.
// ---------------------------------------------------------------------------
template <class T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<_Float16> {
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }  // to nearest even
};
template <>
struct Elem<__bf16> {
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }  // to nearest even
};

template <class T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// a record's address as a pointer to global memory (not a generic one, whose
// accesses also go through the LDS counters)
template <class T>
using Glob = __attribute__((address_space(1))) T *;

template <class T>
__device__ __forceinline__ Glob<T> glob(uint64_t base, uint64_t off)
{
    return reinterpret_cast<Glob<T>>(base) + off;
}

template <class T, int V, bool NT = false>
__device__ __forceinline__ typename VecOf<T, V>::type ldv(Glob<const T> p)
{
    const auto v = reinterpret_cast<Glob<const typename VecOf<T, V>::type>>(p);
    return NT ? __builtin_nontemporal_load(v) : *v;
}

template <class T, int V>
__device__ __forceinline__ void stv(Glob<T> p, const float (&v)[V])
{
    typename VecOf<T, V>::type o;
#pragma unroll
    for (int k = 0; k < V; ++k)
        o[k] = Elem<T>::down(v[k]);
    __builtin_nontemporal_store(o, reinterpret_cast<Glob<typename VecOf<T, V>::type>>(p));
}

// one element of a lane's own tensor
__device__ __forceinline__ float ld_any(uint64_t pt, uint64_t off)
{
    const uint32_t type = (uint32_t)(pt >> 56);
    const uint64_t base = pt & 0x00ffffffffffffffull;
    if (type == kTF32)
        return *glob<const float>(base, off);
    const uint16_t h = *glob<const uint16_t>(base, off);
    return type == kTBF16 ? __uint_as_float((uint32_t)h << 16) : (float)__builtin_bit_cast(_Float16, h);
}
__device__ __forceinline__ void st_any(uint64_t pt, uint64_t off, float v)
{
    const uint32_t type = (uint32_t)(pt >> 56);
    const uint64_t base = pt & 0x00ffffffffffffffull;
    if (type == kTF32)
        *glob<float>(base, off) = v;
    else if (type == kTBF16)
        *glob<__bf16>(base, off) = Elem<__bf16>::down(v);
    else
        *glob<_Float16>(base, off) = Elem<_Float16>::down(v);
}

}  // namespace gc
