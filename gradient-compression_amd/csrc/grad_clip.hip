// grad_clip.hip — the global norm of many gradient tensors and the clipping
// that follows it (include/gcodec.h gc_grad_*, gc_qsgd_decode_clip).
//
//   N = (sum_t sum_i |x_ti|^p)^(1/p),  p = 1, 2 or infinity (N = max |x|)
//   c = min(1, max_norm / (N + 1e-6)),  y = RN_type(x c)
//
// Two passes, and nothing is kept between calls: k_grad_norm (or k_lane_norm,
// from packed words) leaves one partial a block in the caller's workspace, and
// the first wave of every block of the pass that writes (k_grad_scale, k_decode_clip)
// adds those partials in one fixed order and forms c.  So there are no atomics, no
// tickets and no zeroed state: the result does not depend on the schedule, a
// captured call owns all that it writes, and two calls on different streams
// share nothing.  A list that one block can read in a few microseconds
// (kOneElems) is done by one block in one launch.
//
// Sums are held in 64 bits: the square of a float32 is exact to half an ulp
// there and cannot overflow or vanish, so N is right for any gradients whose
// norm a float32 can hold (1e-45 .. 3e38) and c even beyond.  One conversion
// and one fused multiply-add for each element are about a seventh of the
// vector unit's time at the rate that the memory delivers float32.
//
// All of it is bound by HBM.  The norm reads the gradients once, clipping reads
// them twice and writes them once; of a list beyond the 256 MB of cache in front
// of the memory, the first read passes all but the end by the cache, and the
// second finds that end there.  Short lists are bound by the two launches and
// the chain partials -> c -> table -> first load inside the second: 10,000 /
// 70,000 / 250,000 / a million float32 take 8.0 / 8.5 / 8.7 / 9.9 us in 3 tensors and
// 12.2 / 9.9 / 9.8 / 11.0 in 500.
#include "gc_device.h"
#include "gc_host.h"
#include "grads.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace gc {

// Flat elements a wave takes at a time, at most: 8 KB of float32 (eight vectors
// a lane).  16-bit lists take twice as many in the norm: 426M bfloat16 139 us
// against 149 at 2048; float32 loses by it (1e9: 588 against 579).
constexpr uint32_t kTile = 2048;
constexpr uint32_t kLeastTile = 256;  // a vector of float32 a lane

// Two blocks a CU, 32 waves of 4 KB in flight each.  256 / 512 / 1024 blocks:
// 18.7 / 17.4 / 18.6 us on 94 MB of float32.
constexpr unsigned kNormThreads = 1024;
constexpr unsigned kNormGrid = 512;

// The pass that writes runs best with about a tile a wave, in small blocks that
// come and go (2048 / 16384 blocks: 474 / 437 us on 426M bfloat16), but where
// most tiles are under way at once, fewer and larger blocks form c fewer times
// (14.7M float32: 33.7 us in blocks of 256, 32.4 in blocks of 1024; at 426M
// elements 387 and 416).  Both passes of a list of up to kSpread tiles go in
// small blocks again, over more CUs (60,000 elements of 3 tensors 8.8 -> 7.9 us).
constexpr unsigned kScaleThreads = 256;
constexpr unsigned kScaleGrid = 16384;
// The waves that 256 CUs hold at most, 32 each.  Blocks of 256 threads of
// k_grad_scale come to half of it: their two tables take 33 KB of a CU's 160 KB of LDS.
constexpr uint64_t kWaves = 8192;
constexpr uint64_t kSpread = 1024;

// Words: one block a CU adds them (128 / 256 / 512 blocks: 33.3 / 30.9 / 32.5 us
// with the decode, whose every block reads the partials).  The decode's grid hardly
// matters (2560 / 4096 / 5120 / 8192 blocks: 254 / 259 / 250 / 249 us for 246M
// bfloat16, 96.4 / 95.3 / 95.1 / 95.2 us for 100M float32): whole rounds, four, of
// the 1280 blocks that are resident at once (90 registers: five a CU).
constexpr unsigned kLaneGrid = 256;
constexpr unsigned kDecodeGrid = 5120;

// What one block does alone (one_block) and the average sizes below which
// tensors count as small: for the sums and the scaling of a list, and for
// each tensor's own norm.
constexpr uint64_t kOneElems = 8192;
constexpr uint64_t kFewElems = 1024;
constexpr uint64_t kFewEach = 64;

// The tensors of a tile beyond which lanes take their own: 3 / 5 for clipping
// 120,000 elements of 500 tensors 12.2 / 13.0 us, for each norm of a million of 300
// 15.5 / 12.0.
constexpr uint32_t kMany = 3;
constexpr uint32_t kManyEach = 5;

// The cache in front of HBM.  Clipping 426M bfloat16 takes 374 us with the last
// 256 MB read through it, 377 with 192, 394 with 320, 404 with none, and 437
// with everything.
constexpr uint64_t kCacheBytes = 256ull << 20;
constexpr double kEps = 1e-6;

// workspace: kNormGrid partials (64-bit), kNormGrid maxima (32-bit), then the
// pieces' sums of the per-tensor norms
constexpr size_t kWsPeak = kNormGrid * 8;
constexpr size_t kWsSlots = kWsPeak + kNormGrid * 4;

// p as the kernels' template argument; kPInf sums by maximum
constexpr int kPInf = 0;

// ---------------------------------------------------------------------------
// accumulation
// ---------------------------------------------------------------------------
// An accumulator of |x|^p.  p = infinity keeps the bits of |x| as an integer:
// their order is the values' order, and a NaN is above them all and stays.
template <int P>
struct Acc {
    double v = 0.0;
    __device__ __forceinline__ void add(float x)
    {
        const double d = (double)x;
        v = P == 2 ? fma(d, d, v) : v + fabs(d);
    }
    __device__ __forceinline__ void join(const Acc &o) { v += o.v; }
    __device__ __forceinline__ Acc shuffled(int m) const
    {
        Acc r;
        r.v = __shfl_xor(v, m, 64);
        return r;
    }
    __device__ __forceinline__ double value() const { return v; }
    __device__ __forceinline__ void set(double x) { v = x; }
};
template <>
struct Acc<kPInf> {
    uint32_t m = 0;
    __device__ __forceinline__ void add(float x) { m = max(m, __float_as_uint(x) & 0x7fffffffu); }
    __device__ __forceinline__ void join(const Acc &o) { m = max(m, o.m); }
    __device__ __forceinline__ Acc shuffled(int k) const
    {
        Acc r;
        r.m = (uint32_t)__shfl_xor((int)m, k, 64);
        return r;
    }
    __device__ __forceinline__ double value() const { return (double)__uint_as_float(m); }
    __device__ __forceinline__ void set(double x) { m = __float_as_uint((float)x); }  // a float's own value back
};

template <class A>
__device__ __forceinline__ void wave_join(A &a)
{
#pragma unroll
    for (int m = 32; m; m >>= 1)
        a.join(a.shuffled(m));
}

// the wave's elements x[0 .. cnt), x and cnt the same for all lanes; NT: past
// the cache (1e9 float32 in 577 us, 6.9 TB/s, against 645 through it)
template <class T, bool NT, class F>
__device__ __forceinline__ void wave_read(Glob<const T> x, uint32_t cnt, F f)
{
    constexpr uint32_t V = 16 / sizeof(T), step = 64 * V, U = 4;
    const uint32_t lane = lane_id();
    uint32_t i = 0;
    for (; i + U * step <= cnt; i += U * step) {
        typename VecOf<T, V>::type v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            v[u] = ldv<T, V, NT>(x + i + u * step + lane * V);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t k = 0; k < V; ++k)
                f(Elem<T>::up(v[u][k]));
    }
    for (; i < cnt; i += step) {
        const uint32_t j = i + lane * V;
        if (j + V <= cnt) {
            const auto v = ldv<T, V>(x + j);
#pragma unroll
            for (uint32_t k = 0; k < V; ++k)
                f(Elem<T>::up(v[k]));
        } else {
            for (uint32_t k = j; k < cnt; ++k)
                f(Elem<T>::up(x[k]));
        }
    }
}

template <bool NT, class F>
__device__ __forceinline__ void wave_read_any(uint32_t type, uint64_t base, uint64_t off, uint32_t cnt, F f)
{
    if (type == kTF32)
        wave_read<float, NT>(glob<const float>(base, off), cnt, f);
    else if (type == kTBF16)
        wave_read<__bf16, NT>(glob<const __bf16>(base, off), cnt, f);
    else
        wave_read<_Float16, NT>(glob<const _Float16>(base, off), cnt, f);
}

// f(i, x) for element lo + i of a tile of kLeastTile or fewer elements of
// tensors s0 .. s1, the lane's own: four lookups, then four loads in flight.
// Clipping 5000 elements of 500 tensors takes 14.3 us so, 83.8 when each tensor
// is waited for.
template <class F>
__device__ __forceinline__ void lane_read(const GradRec *rec, uint32_t s0, uint32_t s1, uint64_t lo, uint64_t hi, F f)
{
    constexpr uint32_t U = kLeastTile / 64;
    float x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint64_t e = lo + u * 64 + lane_id();
        if (e < hi) {
            const uint32_t s = grad_lane(rec, s0, s1, e);
            x[u] = ld_any(rec[s].pt, e - rec[s].start);
        }
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u)
        if (lo + u * 64 + lane_id() < hi)
            f(u * 64 + lane_id(), x[u]);
}

// The share of a block of `per` waves of the sum of |x|^p and (PEAK) of max |x|,
// valid in thread 0; elements ahead of `cold` are read past the cache.
// EACH: also the sum of every piece, at slot (tile + tensor): along the flat
// sequence each next piece has the next tile or the next tensor, so a tensor's
// pieces have consecutive slots of their own.
template <int P, bool EACH, bool PEAK>
__device__ __forceinline__ void block_norm(uint32_t per, const GradRec *rec, uint32_t count, uint64_t n, uint32_t tile,
                                           uint64_t cold, double *__restrict__ slots, Acc<P> &all, Acc<kPInf> &top)
{
    __shared__ double sacc[kNormThreads / 64];
    __shared__ uint32_t smax[kNormThreads / 64];
    __shared__ double svals[EACH ? kNormThreads / 64 : 1][EACH ? kLeastTile : 1];
    const uint64_t waves = (uint64_t)gridDim.x * per;
    for (uint64_t t = (uint64_t)blockIdx.x * per + wave_id(); t * tile < n; t += waves) {
        const uint64_t lo = t * tile, hi = min(lo + tile, n);
        const uint32_t s0 = uni32(grad_find(rec, count, lo));
        if (tile == kLeastTile && grad_many(rec, count, s0, hi, EACH ? kManyEach : kMany)) {
            const uint32_t s1 = uni32(grad_find(rec, count, hi - 1));
            double *v = EACH ? svals[wave_id()] : nullptr;
            lane_read(rec, s0, s1, lo, hi, [&](uint32_t i, float x) {
                Acc<P> one;
                one.add(x);
                all.join(one);
                if (PEAK)
                    top.add(x);
                if (EACH)
                    v[i] = one.value();
            });
            if (EACH) {  // the pieces' sums, a lane a piece, in the elements' order
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
                for (uint32_t s = s0 + lane_id(); s <= s1; s += 64) {
                    const uint64_t a = max(rec[s].start, lo), b = min(rec[s + 1].start, hi);
                    Acc<P> one;
                    for (uint64_t e = a; e < b; e += 8) {  // eight reads in flight; 0 joins without effect
                        double x[8];
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            x[k] = e + k < b ? v[e + k - lo] : 0.0;
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) {
                            Acc<P> o;
                            o.set(x[k]);
                            one.join(o);
                        }
                    }
                    if (a < b)
                        slots[t + s] = one.value();
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
            }
            continue;
        }
        grad_walk(rec, s0, lo, hi,
                  [&](uint32_t s, uint32_t type, uint64_t base, uint64_t start, uint64_t a, uint64_t b) {
                      Acc<P> one;
                      Acc<P> &acc = EACH ? one : all;
                      auto add = [&](float x) {
                          acc.add(x);
                          if (PEAK)
                              top.add(x);
                      };
                      if (lo < cold)
                          wave_read_any<true>(type, base, a - start, (uint32_t)(b - a), add);
                      else
                          wave_read_any<false>(type, base, a - start, (uint32_t)(b - a), add);
                      if (EACH) {
                          all.join(one);
                          wave_join(one);
                          if (lane_id() == 0)
                              slots[t + s] = one.value();
                      }
                  });
    }
    wave_join(all);
    if (PEAK)
        wave_join(top);
    if (lane_id() == 0) {
        sacc[wave_id()] = all.value();
        if (PEAK)
            smax[wave_id()] = top.m;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (unsigned w = 1; w < per; ++w) {
            Acc<P> o;
            o.set(sacc[w]);
            all.join(o);
            if (PEAK)
                top.m = max(top.m, smax[w]);
        }
}

// ---------------------------------------------------------------------------
// finish: the partials in one fixed order, by every wave that needs them
// ---------------------------------------------------------------------------
template <int P>
__device__ __forceinline__ double wave_total(const double *__restrict__ part, uint32_t parts)
{
    constexpr uint32_t U = 8;  // loads in flight: a large tensor has tens of thousands of slots
    Acc<P> a;
    uint32_t i = lane_id();
    for (; i + (U - 1) * 64 < parts; i += U * 64) {
        double v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            v[u] = part[i + u * 64];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            Acc<P> o;
            o.set(v[u]);
            a.join(o);
        }
    }
    for (; i < parts; i += 64) {
        Acc<P> o;
        o.set(part[i]);
        a.join(o);
    }
    wave_join(a);
    return a.value();
}

__device__ __forceinline__ double wave_total_of(int p, const double *part, uint32_t parts)
{
    return p == 2 ? wave_total<2>(part, parts) : p == 1 ? wave_total<1>(part, parts) : wave_total<kPInf>(part, parts);
}

__device__ __forceinline__ double root_of(int p, double total) { return p == 2 ? sqrt(total) : total; }

// min(1, max_norm / (N + 1e-6)); a NaN stays one, as in torch's clamp
__device__ __forceinline__ float clip_coef(double norm, double max_norm)
{
    const double q = max_norm / (norm + kEps);
    return q > 1.0 ? 1.0f : (float)q;
}

__device__ __forceinline__ void write_norm(int p, double t, double *total, float *norm)
{
    if (total)
        *total = t;
    if (norm)
        *norm = (float)root_of(p, t);
}

// the norm of tensor s from its slots; the wave's, or (WAVES > 1) the block's:
// the same number of slots for every wave's share, then the waves in order
template <int P, unsigned WAVES>
__device__ __forceinline__ void tensor_norm(const GradRec *rec, uint32_t s, uint32_t tile, const double *slots,
                                            float *__restrict__ each)
{
    const uint64_t a = uni64(rec[s].start), b = uni64(rec[s + 1].start);
    double t = 0.0;
    if (a != b) {
        const uint64_t s0 = a / tile + s, cnt = (b - 1) / tile + s + 1 - s0;
        const uint64_t share = (cnt + WAVES - 1) / WAVES, w0 = WAVES > 1 ? wave_id() * share : 0;
        t = wave_total<P>(slots + s0 + w0, w0 < cnt ? (uint32_t)min(share, cnt - w0) : 0u);
    }
    if constexpr (WAVES > 1) {
        __shared__ double sw[WAVES];
        if (lane_id() == 0)
            sw[wave_id()] = t;
        __syncthreads();
        if (wave_id() != 0)
            return;
        t = wave_total<P>(sw, WAVES);
    }
    if (lane_id() == 0)
        each[s] = (float)root_of(P, t);
}

// The norm's first pass: one partial a block, or the whole call in one block
// (alone).  A block's tiles are 16 consecutive ones of every gridDim.x * 16,
// so the chip reads a few MB of consecutive addresses at any time.  Bound by
// HBM: 4 GB of float32 in 579 us (6.9 TB/s), 853 MB of bfloat16 in 125 us
// (6.8 TB/s; 132 us with each tensor's norm); 94 MB of float32 in 17 us, of which
// 4 us are the launch and the first loads.
template <int P, bool EACH, bool PEAK, bool LDS>
__global__ __launch_bounds__(kNormThreads, 8) void k_grad_norm(GradArg g, uint64_t n, uint32_t tile, uint64_t cold,
                                                               bool alone, double *__restrict__ part,
                                                               uint32_t *__restrict__ peak, double *slots,
                                                               double *__restrict__ total, float *__restrict__ norm,
                                                               float *__restrict__ each)
{
    __shared__ GradRec srec[LDS ? kLdsRecs + 1 : 1];
    const GradRec *rec = LDS ? srec : g.rec;
    if (LDS && g.count) {
        stage_table(g, srec);
        __syncthreads();
    }
    Acc<P> all;
    Acc<kPInf> top;
    block_norm<P, EACH, PEAK>(blockDim.x >> 6, rec, g.count, n, tile, cold, slots, all, top);
    if (threadIdx.x == 0) {
        if (part)
            part[blockIdx.x] = all.value();
        if (PEAK)
            peak[blockIdx.x] = top.m;
        if (alone)
            write_norm(P, all.value(), total, norm);
    }
    if (EACH && alone)  // behind block_norm's barrier, which the slots' writes are ahead of
        for (uint32_t s = wave_id(); s < g.count; s += blockDim.x >> 6)
            tensor_norm<P, 1>(rec, s, tile, slots, each);
}

// The norm's second pass, over the partials.  Block 0: the total and N; block
// 1 + s: the norm of tensor s.  Latency: 4 us for 512 partials, 6.5 us with each
// norm where the largest tensor has 16,000 slots.
template <int P>
__global__ __launch_bounds__(kNormThreads) void k_grad_finish(GradArg g, uint32_t tile, const double *__restrict__ part,
                                                              uint32_t parts, const double *__restrict__ slots,
                                                              double *__restrict__ total, float *__restrict__ norm,
                                                              float *__restrict__ each)
{
    if (blockIdx.x > 0) {
        tensor_norm<P, kNormThreads / 64>(g.rec, blockIdx.x - 1, tile, slots, each);
    } else if (wave_id() == 0) {
        const double t = wave_total<P>(part, parts);
        if (lane_id() == 0)
            write_norm(P, t, total, norm);
    }
}

// ---------------------------------------------------------------------------
// scale
// ---------------------------------------------------------------------------
template <class TS, class TD, bool NT>
__device__ __forceinline__ void wave_scale(Glob<const TS> x, Glob<TD> y, uint32_t cnt, float c)
{
    constexpr uint32_t V = sizeof(TS) == 2 && sizeof(TD) == 2 ? 8 : 4, step = 64 * V, U = 4;
    const uint32_t lane = lane_id();
    uint32_t i = 0;
    for (; i + U * step <= cnt; i += U * step) {
        typename VecOf<TS, V>::type v[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            v[u] = ldv<TS, V, NT>(x + i + u * step + lane * V);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            float f[V];
#pragma unroll
            for (uint32_t k = 0; k < V; ++k)
                f[k] = Elem<TS>::up(v[u][k]) * c;
            stv<TD, V>(y + i + u * step + lane * V, f);
        }
    }
    for (; i < cnt; i += step) {
        const uint32_t j = i + lane * V;
        if (j + V <= cnt) {
            const auto v = ldv<TS, V>(x + j);
            float f[V];
#pragma unroll
            for (uint32_t k = 0; k < V; ++k)
                f[k] = Elem<TS>::up(v[k]) * c;
            stv<TD, V>(y + j, f);
        } else {
            for (uint32_t k = j; k < cnt; ++k)
                y[k] = Elem<TD>::down(Elem<TS>::up(x[k]) * c);
        }
    }
}

template <class TS, bool NT>
__device__ __forceinline__ void wave_scale_to(uint32_t td, Glob<const TS> x, uint64_t base, uint64_t off, uint32_t cnt,
                                              float c)
{
    if (td == kTF32)
        wave_scale<TS, float, NT>(x, glob<float>(base, off), cnt, c);
    else if (td == kTBF16)
        wave_scale<TS, __bf16, NT>(x, glob<__bf16>(base, off), cnt, c);
    else
        wave_scale<TS, _Float16, NT>(x, glob<_Float16>(base, off), cnt, c);
}

// The tile from element lo on of y = RN(x c), from the tensors of src into those
// of dst (the same sizes), or (FLAT) end to end into float32
template <bool FLAT, bool NT>
__device__ __forceinline__ void scale_tile(const GradRec *rs, const GradRec *rd, uint32_t count, float *flat, uint64_t n,
                                           uint64_t lo, uint32_t tile, float c)
{
    const uint64_t hi = min(lo + tile, n);
    const uint32_t s0 = uni32(grad_find(rs, count, lo));
    if (tile == kLeastTile && grad_many(rs, count, s0, hi, kMany)) {
        const uint32_t s1 = uni32(grad_find(rs, count, hi - 1));
        lane_read(rs, s0, s1, lo, hi, [&](uint32_t i, float x) {
            const uint64_t e = lo + i;
            if (FLAT) {
                flat[e] = x * c;
            } else {
                const uint32_t s = grad_lane(rs, s0, s1, e);
                st_any(rd[s].pt, e - rd[s].start, x * c);
            }
        });
        return;
    }
    grad_walk(rs, s0, lo, hi, [&](uint32_t s, uint32_t type, uint64_t base, uint64_t start, uint64_t a, uint64_t b) {
        const uint64_t dpt = FLAT ? (uint64_t)kTF32 << 56 | reinterpret_cast<uint64_t>(flat) : uni64(rd[s].pt);
        const uint64_t off = a - start, doff = FLAT ? a : off;
        const uint32_t td = (uint32_t)(dpt >> 56), cnt = (uint32_t)(b - a);
        const uint64_t dbase = dpt & 0x00ffffffffffffffull;
        if (type == kTF32)
            wave_scale_to<float, NT>(td, glob<const float>(base, off), dbase, doff, cnt, c);
        else if (type == kTBF16)
            wave_scale_to<__bf16, NT>(td, glob<const __bf16>(base, off), dbase, doff, cnt, c);
        else
            wave_scale_to<_Float16, NT>(td, glob<const _Float16>(base, off), dbase, doff, cnt, c);
    });
}

// Clipping's second pass.  In place with c = 1, as in most steps of a training
// run, nothing is left to do.  Tiles in the order of the norm: backwards, to
// meet the cache's content first, is no faster (426M bfloat16 380 us against 370,
// 23.5M float32 into a bucket 49.8 against 48.5).  Stores pass the cache: through
// it, what the first pass left there is lost (351 -> 382 us, 246M bfloat16 into a
// bucket).  Bound by HBM: 1.7 GB in 248 us (6.9 TB/s, a part from the cache);
// 118 MB of 14.7M float32 in 22 us, 188 MB of 23.5M into a bucket in 31 us.
template <bool FLAT, bool LDS>
__global__ __launch_bounds__(kNormThreads) void k_grad_scale(GradArg src, GradArg dst, float *flat, uint64_t n,
                                                              uint32_t tile, uint64_t cold, int p, double max_norm,
                                                              const double *__restrict__ part,
                                                              uint32_t parts, const uint32_t *__restrict__ peaks,
                                                              bool in_place, float *__restrict__ norm,
                                                              float *__restrict__ peak)
{
    __shared__ GradRec ss[LDS ? kLdsRecs + 1 : 1];
    __shared__ GradRec sd[LDS && !FLAT ? kLdsRecs + 1 : 1];
    __shared__ float sc;
    const GradRec *rs = LDS ? ss : src.rec, *rd = LDS ? sd : dst.rec;
    if (wave_id() == 0) {
        const double N = root_of(p, wave_total_of(p, part, parts));
        const float c0 = clip_coef(N, max_norm);
        if (lane_id() == 0)
            sc = c0;
        if (blockIdx.x == 0) {
            if (FLAT) {
                // max |RN(x c)| = RN(max |x| c): rounding keeps the order.  A NaN
                // or infinite x with c = NaN or 0 gives NaN on both sides.
                Acc<kPInf> top;
                for (uint32_t i = lane_id(); i < parts; i += 64)
                    top.m = max(top.m, peaks[i]);
                wave_join(top);
                if (lane_id() == 0)
                    *peak = __uint_as_float(top.m) * c0;
            }
            if (norm && lane_id() == 0)
                *norm = (float)N;
        }
    }
    if (LDS && n) {
        stage_table(src, ss);
        if (!FLAT)
            stage_table(dst, sd);
    }
    __syncthreads();
    const float c = sc;
    if (in_place && c == 1.0f)
        return;
    const uint32_t per = blockDim.x >> 6;
    const uint64_t tiles = (n + tile - 1) / tile, waves = (uint64_t)gridDim.x * per;
    for (uint64_t t = (uint64_t)blockIdx.x * per + wave_id(); t < tiles; t += waves) {
        const uint64_t lo = t * tile;
        if (lo < cold)
            scale_tile<FLAT, true>(rs, rd, src.count, flat, n, lo, tile, c);
        else
            scale_tile<FLAT, false>(rs, rd, src.count, flat, n, lo, tile, c);
    }
}

// Both passes in one block, without a second launch: 5.6 us for 1000 elements
// of 3 tensors.  Latency of two rounds of loads.
template <int P, bool FLAT>
__global__ __launch_bounds__(kNormThreads) void k_grad_clip_one(GradArg src, GradArg dst, float *flat, uint64_t n,
                                                                uint32_t tile, double max_norm, bool in_place,
                                                                float *__restrict__ norm, float *__restrict__ peak)
{
    __shared__ GradRec ss[kLdsRecs + 1];
    __shared__ GradRec sd[FLAT ? 1 : kLdsRecs + 1];
    __shared__ float sc;
    if (n) {
        stage_table(src, ss);
        if (!FLAT)
            stage_table(dst, sd);
        __syncthreads();
    }
    Acc<P> all;
    Acc<kPInf> top;
    block_norm<P, false, FLAT>(kNormThreads / 64, ss, src.count, n, tile, 0, nullptr, all, top);
    if (threadIdx.x == 0) {
        const double N = root_of(P, all.value());
        sc = clip_coef(N, max_norm);
        if (norm)
            *norm = (float)N;
        if (FLAT)
            *peak = __uint_as_float(top.m) * sc;
    }
    __syncthreads();
    const float c = sc;
    if (in_place && c == 1.0f)
        return;
    for (uint64_t lo = (uint64_t)wave_id() * tile; lo < n; lo += (uint64_t)(kNormThreads / 64) * tile)
        scale_tile<FLAT, false>(ss, sd, src.count, flat, n, lo, tile, c);
}

// ---------------------------------------------------------------------------
// decode: v = RN(RN(k Q) alpha), k = RN(norm / s), Q = lane - W s (k_qsgd_decode's
// arithmetic), the norm of the v, and y = RN_type(RN(v c))
// ---------------------------------------------------------------------------
struct LaneArg {
    const uint32_t *words;
    uint64_t n, M;
    const float *norm;
    float s, alpha;
    int32_t sub;   // W s
    uint32_t w;    // lane width
    uint32_t L;    // lanes a word
    uint32_t qmax; // largest |Q|
    uint64_t cold; // words the norm reads past the cache
    uint32_t split; // shares of a tile's planes
};

// v depends on Q alone, so the norm is |k alpha| times the norm of the
// integers, whose sum is exact in any order.  Where that product is not the
// sum of the rounded v to within their own roundings (values that overflow or
// fall below the normal range, wide lanes whose squares pass 32 bits), the
// values themselves are added in 64 bits.
__device__ __forceinline__ bool lanes_exact(const LaneArg &a, float k)
{
    const double step = fabs((double)k * (double)a.alpha), top = fabs((double)k) * (double)a.qmax;
    return a.w <= 14 && step >= 1e-30 && step <= 1e30 && top <= 1e38 && top * fabs((double)a.alpha) <= 1e38;
}

// A partial is the exact integer sum, or the bits of the 64-bit sum of values
template <int P>
__device__ __forceinline__ uint64_t lanes_join(bool exact, uint64_t x, uint64_t y)
{
    if (exact)
        return P == kPInf ? max(x, y) : x + y;
    Acc<P> a, b;
    a.set(__longlong_as_double((long long)x));
    b.set(__longlong_as_double((long long)y));
    a.join(b);
    return (uint64_t)__double_as_longlong(a.value());
}

template <int P>
__device__ __forceinline__ uint64_t lanes_wave(bool exact, uint64_t x)
{
#pragma unroll
    for (int m = 32; m; m >>= 1)
        x = lanes_join<P>(exact, x, __shfl_xor(x, m, 64));
    return x;
}

template <int P>
__device__ __forceinline__ double lanes_root(const LaneArg &a, float k, bool exact, uint64_t t)
{
    if (!exact)
        return root_of(P, __longlong_as_double((long long)t));
    if (P == kPInf)
        return fabs((double)(k * (float)t * a.alpha));
    const double step = fabs((double)k * (double)a.alpha);
    return P == 2 ? step * sqrt((double)t) : step * (double)t;
}

// four words' lanes l0 <= l < l1 at flat elements l M + i .. + 3; CHECK: those below n
template <int P, bool CHECK>
__device__ __forceinline__ uint32_t quad_sum(const LaneArg &a, uint4 wd, uint64_t i, uint32_t l0, uint32_t l1,
                                             uint32_t mask, uint32_t sum)
{
    for (uint32_t l = l0; l < l1; ++l) {
        const uint32_t we[4] = {wd.x, wd.y, wd.z, wd.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int32_t q = (int32_t)((we[e] >> (l * a.w)) & mask) - a.sub;  // |q| < 2^14
            if (CHECK && (uint64_t)l * a.M + i + e >= a.n)
                q = 0;
            if (P == 2) {
                sum += (uint32_t)__mul24(q, q);
            } else {
                const uint32_t m = (uint32_t)(q < 0 ? -q : q);
                sum = P == kPInf ? max(sum, m) : sum + m;
            }
        }
    }
    return sum;
}

__device__ __forceinline__ uint4 ld_nt4u(const uint4 *p)
{
    typedef uint32_t u4v __attribute__((ext_vector_type(4)));
    const u4v v = __builtin_nontemporal_load(reinterpret_cast<const u4v *>(p));
    return make_uint4(v.x, v.y, v.z, v.w);
}

// the block's share of the norm of the words, valid in thread 0
template <int P>
__device__ __forceinline__ uint64_t block_lanes(const LaneArg &a, float k, bool exact)
{
    __shared__ uint64_t part[kNormThreads / 64];
    const uint32_t mask = a.w >= 32 ? 0xffffffffu : (1u << a.w) - 1u;
    const uint32_t full = (uint32_t)min(a.M ? a.n / a.M : 0, (uint64_t)a.L);  // planes that are full to the end
    const uint64_t quads = a.M >> 2, stride = (uint64_t)gridDim.x * kNormThreads;
    const uint4 *words = reinterpret_cast<const uint4 *>(a.words);
    uint64_t t = (uint64_t)blockIdx.x * kNormThreads + threadIdx.x, sum = 0;
    if (exact) {
        // w <= 14: a quad's sum is at most L * 4 * 2^(2w) <= 2^31
        auto add = [&](uint4 wd, uint64_t i) {
            uint32_t q = quad_sum<P, false>(a, wd, i, 0, full, mask, 0u);
            q = quad_sum<P, true>(a, wd, i, full, a.L, mask, q);
            sum = lanes_join<P>(true, sum, (uint64_t)q);
        };
        constexpr int U = 4;  // loads in flight, also for the last quads
        for (; t < quads; t += U * stride) {
            uint4 wd[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t j = min(t + u * stride, quads - 1);
                wd[u] = 4 * j < a.cold ? ld_nt4u(words + j) : words[j];
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (t + u * stride < quads)
                    add(wd[u], 4 * (t + u * stride));
        }
    } else {
        Acc<P> real;
        for (; t < quads; t += stride) {
            const uint4 wd = words[t];
            const uint32_t we[4] = {wd.x, wd.y, wd.z, wd.w};
            for (uint32_t l = 0; l < a.L; ++l)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int32_t q = (int32_t)((we[e] >> (l * a.w)) & mask) - a.sub;
                    if ((uint64_t)l * a.M + 4 * t + e < a.n)
                        real.add(k * (float)q * a.alpha);
                }
        }
        sum = (uint64_t)__double_as_longlong(real.value());
    }
    sum = lanes_wave<P>(exact, sum);
    if (lane_id() == 0)
        part[wave_id()] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        for (unsigned w = 1; w < kNormThreads / 64; ++w)
            sum = lanes_join<P>(exact, sum, part[w]);
    return sum;
}

// The words' first pass: 1/6 (4 bit, one rank) to 1/2 (8 bit, eight ranks) of what
// reading the decoded float32 gradients would take.  Bound by HBM where there are many
// (491 MB in 75 us, 6.5 TB/s); 15.7 MB take 8 us, half of it the launch and the
// first loads.
template <int P>
__global__ __launch_bounds__(kNormThreads) void k_lane_norm(LaneArg a, uint64_t *__restrict__ part)
{
    const float k = *a.norm / a.s;
    const uint64_t sum = block_lanes<P>(a, k, lanes_exact(a, k));
    if (threadIdx.x == 0)
        part[blockIdx.x] = sum;
}

// the lane's quad v of flat elements i .. i + 3, those inside [a, b), to the
// tensor at base whose first element is start
template <class T>
__device__ __forceinline__ void store_quad(uint64_t base, uint64_t start, uint64_t a, uint64_t b, uint64_t i,
                                           const float (&v)[4])
{
    const Glob<T> y = glob<T>(base, 0);
    if (i >= a && i + 4 <= b) {
        stv<T, 4>(y + (i - start), v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e >= a && i + e < b)
            y[i + e - start] = Elem<T>::down(v[e]);
}

// A unit is planes l0 .. l1 - 1 of a tile of 256 kQuads consecutive words: of
// each plane a range of as many flat elements.  Its words are loaded apart from
// their use, ahead of what the block waits for.
constexpr int kQuads = 2;
struct Unit {
    uint64_t j0;
    uint32_t l0, l1;
    uint4 wd[kQuads];
};

__host__ __device__ __forceinline__ uint64_t decode_tiles(uint64_t M) { return (M + 256 * kQuads - 1) / (256 * kQuads); }

__device__ __forceinline__ Unit decode_load(const LaneArg &a, uint64_t u)
{
    Unit x;
    const uint32_t per = (a.L + a.split - 1) / a.split;
    x.j0 = u / a.split * (256 * kQuads);
    x.l0 = (uint32_t)(u % a.split) * per;
    x.l1 = min(x.l0 + per, a.L);
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        const uint64_t j = x.j0 + 256 * q + 4 * lane_id();  // M is a multiple of 4: a quad is in or out
        x.wd[q] = j < a.M ? *reinterpret_cast<const uint4 *>(a.words + j) : make_uint4(0, 0, 0, 0);
    }
    return x;
}

struct DecodeArg {
    float k, alpha, c;
    int32_t sub;
    uint32_t mask;
};

__device__ __forceinline__ void decode_quad(const DecodeArg &d, uint4 wd, uint32_t sh, float (&v)[4])
{
    const uint32_t we[4] = {wd.x, wd.y, wd.z, wd.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int32_t Q = (int32_t)((we[e] >> sh) & d.mask) - d.sub;
        const float t = d.k * (float)Q;
        v[e] = t * d.alpha * d.c;
    }
}

template <class T>
__device__ __forceinline__ void decode_whole(const DecodeArg &d, const Unit &x, uint32_t sh, Glob<T> y)
{
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        float v[4];
        decode_quad(d, x.wd[q], sh, v);
        stv<T, 4>(y + (256 * q + 4 * lane_id()), v);
    }
}

// Issue bound until the lookups were shared out (30.3 us for ResNet50's 23.5M at
// 4 bits, 28.4 since): lane l finds plane l0 + l's tensor (at most 32 planes),
// all at once, and a plane that lies whole in one tensor is written without a
// test.  A range of many tensors is written lane by lane (1000 elements of 480
// tensors 22 -> 7 us).
__device__ __forceinline__ void decode_unit(const LaneArg &a, const GradRec *rd, uint32_t count, const Unit &x, float k,
                                            float c)
{
    constexpr uint32_t kWords = 256 * kQuads;
    const DecodeArg d{k, a.alpha, c, a.sub, a.w >= 32 ? 0xffffffffu : (1u << a.w) - 1u};
    const uint32_t lane = lane_id();
    if (x.l0 >= x.l1 || (uint64_t)x.l0 * a.M + x.j0 >= a.n)
        return;
    const uint64_t first = (uint64_t)min(x.l0 + lane, x.l1 - 1) * a.M + x.j0;
    const uint32_t mine = x.l1 - x.l0 == 1 ? grad_find(rd, count, first)
                          : first < a.n    ? grad_lane(rd, 0, count - 1, first)
                                           : 0;
    const uint64_t mpt = rd[mine].pt, mstart = rd[mine].start, mend = rd[mine + 1].start;
    const uint32_t len = (uint32_t)min((uint64_t)kWords, a.M - x.j0);
    for (uint32_t l = x.l0; l < x.l1; ++l) {
        const uint64_t lo = (uint64_t)l * a.M + x.j0, hi = min(lo + len, a.n);
        if (lo >= hi)
            break;
        const int at = (int)(l - x.l0);
        auto of = [&](uint64_t v) {
            return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), at) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, at);
        };
        const uint64_t pt = of(mpt), start = of(mstart), end = of(mend);
        const uint32_t sh = l * a.w;
        if (hi <= end && hi - lo == kWords) {
            const uint64_t base = pt & 0x00ffffffffffffffull;
            const uint32_t type = (uint32_t)(pt >> 56);
            if (type == kTF32)
                decode_whole<float>(d, x, sh, glob<float>(base, lo - start));
            else if (type == kTBF16)
                decode_whole<__bf16>(d, x, sh, glob<__bf16>(base, lo - start));
            else
                decode_whole<_Float16>(d, x, sh, glob<_Float16>(base, lo - start));
            continue;
        }
        const uint32_t s0 = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
        if (grad_many(rd, count, s0, hi, kMany)) {
            const uint32_t s1 = uni32(grad_find(rd, count, hi - 1));
#pragma unroll
            for (int q = 0; q < kQuads; ++q) {
                float v[4];
                decode_quad(d, x.wd[q], sh, v);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint64_t i = lo + 256 * q + 4 * lane + e;
                    if (i < hi) {
                        const uint32_t s = grad_lane(rd, s0, s1, i);
                        st_any(rd[s].pt, i - rd[s].start, v[e]);
                    }
                }
            }
            continue;
        }
        grad_walk(rd, s0, lo, hi,
                  [&](uint32_t, uint32_t type, uint64_t base, uint64_t tstart, uint64_t pa, uint64_t pb) {
#pragma unroll
                      for (int q = 0; q < kQuads; ++q) {
                          if (lo + 256 * q >= pb || lo + 256 * (q + 1) <= pa)
                              continue;
                          float v[4];
                          decode_quad(d, x.wd[q], sh, v);
                          const uint64_t i = lo + 256 * q + 4 * lane;
                          if (type == kTF32)
                              store_quad<float>(base, tstart, pa, pb, i, v);
                          else if (type == kTBF16)
                              store_quad<__bf16>(base, tstart, pa, pb, i, v);
                          else
                              store_quad<_Float16>(base, tstart, pa, pb, i, v);
                      }
                  });
    }
}

// The words' second pass: the gradients are written once, clipped.  A thread
// holds two quads of words and writes them plane by plane, so every access of a
// wave is 1 KB (float32) or 512 bytes of consecutive addresses.  Bound by HBM
// for many (491 MB in and 491 MB out in 175 us, 5.6 TB/s); 23.5M float32 at
// 4 bits, 110 MB, take 20 us, of which 5 are the launch and the chain to c.
template <int P, bool LDS>
__global__ __launch_bounds__(kScaleThreads) void k_decode_clip(LaneArg a, GradArg dst, double max_norm,
                                                               const uint64_t *__restrict__ part, uint32_t parts,
                                                               float *__restrict__ norm)
{
    __shared__ GradRec sd[LDS ? kLdsRecs + 1 : 1];
    __shared__ float sc;
    const GradRec *rd = LDS ? sd : dst.rec;
    const uint64_t units = decode_tiles(a.M) * a.split, waves = (uint64_t)gridDim.x * (kScaleThreads / 64);
    uint64_t u = (uint64_t)blockIdx.x * (kScaleThreads / 64) + wave_id();
    Unit x;
    if (u < units)
        x = decode_load(a, u);
    const float k = *a.norm / a.s;
    if (wave_id() == 0) {
        const bool exact = lanes_exact(a, k);
        uint64_t sum = 0;  // the bits of 0.0 as well
        for (uint32_t i = lane_id(); i < parts; i += 64)
            sum = lanes_join<P>(exact, sum, part[i]);
        const double N = lanes_root<P>(a, k, exact, lanes_wave<P>(exact, sum));
        if (lane_id() == 0) {
            sc = clip_coef(N, max_norm);
            if (blockIdx.x == 0)
                *norm = (float)N;
        }
    }
    if (LDS && a.n)
        stage_table(dst, sd);
    __syncthreads();
    const float c = sc;
    while (u < units) {
        decode_unit(a, rd, dst.count, x, k, c);
        u += waves;
        if (u < units)
            x = decode_load(a, u);
    }
}

// both passes in one block
template <int P>
__global__ __launch_bounds__(kNormThreads) void k_decode_clip_one(LaneArg a, GradArg dst, double max_norm,
                                                                  float *__restrict__ norm)
{
    __shared__ GradRec sd[kLdsRecs + 1];
    __shared__ float sc;
    const float k = *a.norm / a.s;
    const bool exact = lanes_exact(a, k);
    if (a.n)
        stage_table(dst, sd);  // ahead of block_lanes's barrier
    const uint64_t sum = block_lanes<P>(a, k, exact);
    if (threadIdx.x == 0) {
        const double N = lanes_root<P>(a, k, exact, sum);
        sc = clip_coef(N, max_norm);
        *norm = (float)N;
    }
    __syncthreads();
    for (uint64_t u = wave_id(), units = decode_tiles(a.M) * a.split; u < units; u += kNormThreads / 64)
        decode_unit(a, sd, dst.count, decode_load(a, u), k, sc);
}

// ---------------------------------------------------------------------------
// table
// ---------------------------------------------------------------------------
constexpr uint32_t kFillRecs = 224;  // records a launch carries in its arguments (3.5 KB)
struct FillArg {
    GradRec rec[kFillRecs];
};

__global__ __launch_bounds__(256) void k_grads_fill(FillArg a, uint32_t cnt, GradRec *__restrict__ out)
{
    if (threadIdx.x < cnt)
        out[threadIdx.x] = a.rec[threadIdx.x];
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static size_t elem_size(uint64_t pt) { return (pt >> 56) == kTF32 ? 4 : 2; }

struct Span {  // a tensor's bytes
    uint64_t lo, hi;
};
static Span span_of(const gc_grads *g, uint64_t s)
{
    const uint64_t pt = g->host_rec[2 * s], lo = pt & 0x00ffffffffffffffull;
    return {lo, lo + (g->host_rec[2 * s + 3] - g->host_rec[2 * s + 1]) * elem_size(pt)};
}

static int check_grads(const gc_grads *g, const char *what)
{
    GC_REQUIRE(g, "%s: null gradient table", what);
    GC_REQUIRE(g->count < (1ull << 31), "%s: more than 2^31 tensors", what);
    GC_REQUIRE(g->host_rec && g->order, "%s: gradient table without its host image", what);
    GC_REQUIRE(g->host_rec[2 * g->count + 1] == g->n, "%s: gradient table's host image does not end at n", what);
    GC_REQUIRE(g->count == 0 || g->rec, "%s: gradient table not on the device", what);
    return GC_OK;
}

static int check_output(const gc_grads *g, const char *what)
{
    GC_REQUIRE(!(g->flags & GC_GRADS_OVERLAP), "%s: tensors to be written share memory", what);
    return GC_OK;
}

// whether [lo, hi) meets a tensor of the table; *at the first one's index
static bool meets(const gc_grads *g, Span x, uint64_t *at)
{
    if (x.lo >= x.hi)
        return false;
    if (g->flags & GC_GRADS_OVERLAP) {  // a later tensor may end ahead of an earlier one
        for (uint64_t s = 0; s < g->count; ++s) {
            const Span y = span_of(g, s);
            if (y.lo < y.hi && y.lo < x.hi && x.lo < y.hi) {
                *at = s;
                return true;
            }
        }
        return false;
    }
    uint64_t a = 0, b = g->count;  // order[]: non-empty tensors by address, then the empty ones
    while (a < b) {
        const uint64_t m = (a + b) / 2;
        const Span y = span_of(g, g->order[m]);
        if (y.lo < y.hi && y.hi <= x.lo)
            a = m + 1;
        else
            b = m;
    }
    if (a == g->count)
        return false;
    const Span y = span_of(g, g->order[a]);
    *at = g->order[a];
    return y.lo < y.hi && y.lo < x.hi;
}

// A tensor may be clipped onto itself; any other input that meets an output
// could be read after it is written.  Both lists by address: one pass.
static int check_apart(const gc_grads *src, const gc_grads *dst, const char *what)
{
    uint64_t j = 0;
    for (uint64_t i = 0; i < src->count; ++i) {
        const uint32_t s = src->order[i];
        const Span x = span_of(src, s);
        if (x.lo >= x.hi)
            break;
        while (j < dst->count) {  // the first output that ends behind x.lo (inputs are by their starts)
            const Span y = span_of(dst, dst->order[j]);
            if (y.lo >= y.hi || y.hi > x.lo)
                break;
            ++j;
        }
        for (uint64_t k = j; k < dst->count; ++k) {
            const uint32_t d = dst->order[k];
            const Span y = span_of(dst, d);
            if (y.lo >= y.hi || y.lo >= x.hi)
                break;
            GC_REQUIRE(s == d && src->host_rec[2 * s] == dst->host_rec[2 * s],
                       "%s: input tensor %u shares memory with output tensor %u", what, s, d);
        }
    }
    return GC_OK;
}

// Memory that a call uses beside its tensors
struct Side {
    const char *name;
    const void *at;  // null: not used
    uint64_t bytes;
    bool written;
};

// Blocks that are done write norms, totals and the output while others still read:
// what a call writes shares memory with nothing else that it uses.
template <size_t N>
static int check_sides(const Side (&side)[N], const gc_grads *src, const gc_grads *dst, const char *what)
{
    for (size_t i = 0; i < N; ++i) {
        const uint64_t lo = reinterpret_cast<uint64_t>(side[i].at);
        const Span x{lo, side[i].at ? lo + side[i].bytes : lo};
        if (x.lo == x.hi)
            continue;
        for (size_t j = i + 1; j < N; ++j) {
            const uint64_t at = reinterpret_cast<uint64_t>(side[j].at);
            const bool apart = !at || side[j].bytes == 0 || at >= x.hi || at + side[j].bytes <= x.lo;
            GC_REQUIRE(apart || !(side[i].written || side[j].written), "%s: %s and %s share memory", what,
                       side[i].name, side[j].name);
        }
        uint64_t at = 0;
        GC_REQUIRE(!(src && side[i].written && meets(src, x, &at)), "%s: %s shares memory with input tensor %llu", what,
                   side[i].name, (unsigned long long)at);
        GC_REQUIRE(!(dst && meets(dst, x, &at)), "%s: %s shares memory with output tensor %llu", what, side[i].name,
                   (unsigned long long)at);
    }
    return GC_OK;
}

static int check_p(uint32_t p, const char *what)
{
    GC_REQUIRE(p == 1 || p == 2 || p == GC_NORM_INF, "%s: the norm is GC_NORM_INF, 1 or 2, got %u", what, p);
    return GC_OK;
}

static int check_max_norm(double m, const char *what)
{
    GC_REQUIRE(m >= 0.0, "%s: max_norm %g is not a number at or above 0", what, m);
    return GC_OK;
}

static GradArg arg_of(const gc_grads *g)
{
    return {reinterpret_cast<const GradRec *>(g->rec), (uint32_t)g->count};
}

// the bytes of the gradients
static uint64_t held_bytes(const gc_grads *g)
{
    uint64_t wide = 0;
    for (uint64_t s = 0; s < g->count; ++s)
        if (elem_size(g->host_rec[2 * s]) == 4)
            wide += g->host_rec[2 * s + 3] - g->host_rec[2 * s + 1];
    return 2 * (g->n + wide);
}

// The elements of a wave's tile: `most`, or as few as spread a short list over
// the chip (over the waves of the one block that does all of it); the least for
// tensors that are small on the whole, which a lane at a time takes.  That goes by
// the list's average: a run of tiny tensors in a list that is large on the whole is
// walked a tensor at a time (clipping 50M elements and 2000 tensors of one takes
// 2.0 ms, 90 us as one tensor; their norm 0.76 ms and 32 us).  Halved
// while the list has less than 16384 of the smaller tiles, but to 256 only below
// 4096 (2M float32: clip 12.7 us at 512, 15.1 at 256; 7M 20.8 at 512, 21.9 at 1024;
// 12M: norm 12.5 at 1024, 15.2 at 2048) and, for 16-bit norms, to 2048 and 1024
// below 32768 (20M: 13.5 us at 1024, 16.3 at 2048).
static uint32_t tile_of(uint64_t n, uint64_t count, uint32_t most, uint64_t few = kFewElems)
{
    if (n < few * count)
        return kLeastTile;
    uint32_t tile = most;
    while (tile > kLeastTile) {
        const uint32_t half = tile / 2;
        const uint64_t want = n <= kOneElems                   ? kNormThreads / 64
                              : half == kLeastTile             ? kWaves / 2
                              : most > kTile && half >= 1024   ? 4 * kWaves
                                                               : 2 * kWaves;
        if (n > half * want)
            break;
        tile = half;
    }
    return tile;
}

// Whether one block does all of a call: a second launch costs 2 us, a tensor
// about what eight elements do.  Clipping 5000 elements of 3 / 60 / 500 tensors
// takes 6.3 / 11.6 / 18.3 us in one block and 8.3 / 11.1 / 13.4 us in two
// launches, 20000 of 3 / 60 tensors 8.8 / 19.2 and 9.5 / 11.1 us.
// Each tensor's own norm: four times that (5000 elements of 300 tensors 23.6 us in
// one block, 14 in two launches).
static bool one_block(uint64_t n, uint64_t count, bool each = false)
{
    return n + (each ? 32 : 8) * count <= kOneElems;
}
static_assert(kOneElems / 8 <= kLdsRecs, "one block's table is in LDS");

// The norm's tile: up to 8 KB of gradients.  Each tensor's own norm takes a
// lane a tensor there, one element after the other, so only the smallest.
static uint32_t norm_tile(const gc_grads *g, bool each = false)
{
    return tile_of(g->n, g->count, held_bytes(g) < 3 * g->n ? 2 * kTile : kTile, each ? kFewEach : kFewElems);
}

// Threads a block for `tiles` tiles: a short list is spread over more CUs
static unsigned norm_threads(uint64_t n, uint64_t count, uint32_t tile, bool each = false)
{
    return !one_block(n, count, each) && n <= (uint64_t)kSpread * tile ? kScaleThreads : kNormThreads;
}

static unsigned norm_grid(uint64_t n, uint64_t count, uint32_t tile, bool each = false)
{
    const uint64_t tiles = (n + tile - 1) / tile, per = norm_threads(n, count, tile, each) / 64;
    if (one_block(n, count, each))
        return 1;
    return (unsigned)std::min<uint64_t>(std::max<uint64_t>((tiles + per - 1) / per, 1), kNormGrid);
}

// of `of` elements or words that take `bytes`, those ahead of the last kCacheBytes
static uint64_t cold_part(uint64_t of, uint64_t bytes)
{
    return bytes <= kCacheBytes ? 0 : (uint64_t)((double)(bytes - kCacheBytes) / (double)bytes * (double)of);
}
static uint64_t cold_elems(const gc_grads *g) { return cold_part(g->n, held_bytes(g)); }

// shares of the planes for which `tiles` tiles of words keep the chip's waves busy
static uint32_t split_of(uint64_t tiles, uint32_t L)
{
    const uint64_t want = kWaves / 2;
    return tiles >= want ? 1u : (uint32_t)std::min<uint64_t>(L, (want + tiles - 1) / std::max<uint64_t>(tiles, 1));
}

static int check_workspace(const gc_grads *g, bool each, const void *workspace, const char *what)
{
    GC_REQUIRE(workspace || gc_grad_workspace_size(g->n, g->count, each) == 0, "%s: null workspace", what);
    GC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7u) == 0, "%s: misaligned workspace", what);
    return GC_OK;
}

static Side workspace_side(const gc_grads *g, bool each, const void *workspace)
{
    return {"the workspace", workspace, gc_grad_workspace_size(g->n, g->count, each), true};
}

// f(p as a constant)
template <class F>
static void with_p(uint32_t p, F f)
{
    if (p == 2)
        f(std::integral_constant<int, 2>());
    else if (p == 1)
        f(std::integral_constant<int, 1>());
    else
        f(std::integral_constant<int, kPInf>());
}

template <bool EACH, bool PEAK>
static void launch_norm(const gc_grads *g, uint32_t p, uint64_t cold, void *ws, double *total, float *norm, float *each,
                        hipStream_t st)
{
    const GradArg a = arg_of(g);
    const uint32_t tile = norm_tile(g, EACH);
    const bool alone = one_block(g->n, g->count, EACH);
    const dim3 grid(norm_grid(g->n, g->count, tile, EACH)), block(norm_threads(g->n, g->count, tile, EACH));
    char *w = alone && !EACH ? nullptr : static_cast<char *>(ws);  // one block leaves no partials
    double *part = reinterpret_cast<double *>(w);
    uint32_t *peak = w ? reinterpret_cast<uint32_t *>(w + kWsPeak) : nullptr;
    double *slots = w ? reinterpret_cast<double *>(w + kWsSlots) : nullptr;
    with_p(p, [&](auto P) {
        if (g->count <= kLdsRecs)
            hipLaunchKernelGGL((k_grad_norm<P(), EACH, PEAK, true>), grid, block, 0, st, a, g->n, tile, cold, alone,
                               part, peak, slots, total, norm, each);
        else
            hipLaunchKernelGGL((k_grad_norm<P(), EACH, PEAK, false>), grid, block, 0, st, a, g->n, tile, cold, alone,
                               part, peak, slots, total, norm, each);
    });
}

static unsigned grid_of(uint64_t tiles, unsigned threads, unsigned most)
{
    const uint64_t per = threads / 64;
    return (unsigned)std::min<uint64_t>(std::max<uint64_t>((tiles + per - 1) / per, 1), most);
}

// threads a block of the scale: large blocks, and so fewer first steps (the
// partials, the table), where most tiles are under way at once; a short list is
// spread over more CUs
static unsigned scale_threads(uint64_t tiles)
{
    return tiles > kSpread && tiles <= 2 * kWaves ? kNormThreads : kScaleThreads;
}

}  // namespace gc

using namespace gc;

static_assert(sizeof(GradRec) == 16, "gc_grads.rec layout");

extern "C" {

int gc_grads_plan(const uint64_t *sizes, const void *const *ptrs, const uint32_t *types, uint64_t count,
                  uint64_t *rec, uint32_t *order, gc_grads *out)
{
    const char *what = "gc_grads_plan";
    GC_REQUIRE(out && rec && order, "%s: null output", what);
    GC_REQUIRE(count == 0 || (sizes && ptrs && types), "%s: null input", what);
    GC_REQUIRE(count < (1ull << 31), "%s: more than 2^31 tensors", what);
    uint64_t n = 0;
    for (uint64_t s = 0; s < count; ++s) {
        GC_REQUIRE(types[s] == GC_F32 || types[s] == GC_F16 || types[s] == GC_BF16,
                   "%s: tensor %llu is not float32, float16 or bfloat16", what, (unsigned long long)s);
        const uint64_t at = reinterpret_cast<uint64_t>(ptrs[s]), size = types[s] == GC_F32 ? 4 : 2;
        GC_REQUIRE(sizes[s] == 0 || ptrs[s], "%s: tensor %llu has no data pointer", what, (unsigned long long)s);
        GC_REQUIRE(at % size == 0 && at >> 56 == 0, "%s: tensor %llu is not aligned to its elements", what,
                   (unsigned long long)s);
        GC_REQUIRE(sizes[s] < (1ull << 52) && n + sizes[s] < (1ull << 52), "%s: size overflow", what);
        const uint64_t tag = types[s] == GC_F32 ? kTF32 : types[s] == GC_F16 ? kTF16 : kTBF16;
        rec[2 * s] = tag << 56 | at;
        rec[2 * s + 1] = n;
        n += sizes[s];
        order[s] = (uint32_t)s;
    }
    rec[2 * count] = 0;
    rec[2 * count + 1] = n;
    gc_grads g{};
    g.count = count;
    g.n = n;
    g.host_rec = rec;
    g.order = order;
    std::sort(order, order + count, [&](uint32_t x, uint32_t y) {
        const Span a = span_of(&g, x), b = span_of(&g, y);
        const bool ea = a.lo == a.hi, eb = b.lo == b.hi;
        if (ea != eb)
            return eb;
        return ea ? x < y : a.lo != b.lo ? a.lo < b.lo : x < y;
    });
    uint64_t end = 0;
    for (uint64_t i = 0; i < count; ++i) {
        const Span a = span_of(&g, order[i]);
        if (a.lo == a.hi)
            break;
        if (a.lo < end)
            g.flags |= GC_GRADS_OVERLAP;
        end = std::max(end, a.hi);
    }
    *out = g;
    return GC_OK;
}

int gc_grads_fill(const gc_grads *grads, uint64_t *rec, gc_stream_t stream)
{
    const char *what = "gc_grads_fill";
    GC_REQUIRE(grads && grads->host_rec && rec, "%s: null pointer", what);
    const GradRec *h = reinterpret_cast<const GradRec *>(grads->host_rec);
    GradRec *d = reinterpret_cast<GradRec *>(rec);
    for (uint64_t i = 0; i <= grads->count; i += kFillRecs) {
        const uint32_t cnt = (uint32_t)std::min<uint64_t>(kFillRecs, grads->count + 1 - i);
        FillArg a;
        std::copy(h + i, h + i + cnt, a.rec);
        std::fill(a.rec + cnt, a.rec + kFillRecs, GradRec{0, 0});
        hipLaunchKernelGGL(k_grads_fill, dim3(1), dim3(256), 0, as_stream(stream), a, cnt, d + i);
    }
    return launch_status(what);
}

size_t gc_grad_workspace_size(uint64_t n, uint64_t count, int each)
{
    if (!each && one_block(n, count))
        return 0;
    // a slot for every piece: at most the tiles and the tensors, of whichever tile the types ask for
    const uint32_t tile = std::min(tile_of(n, count, kTile, kFewEach), tile_of(n, count, 2 * kTile, kFewEach));
    return kWsSlots + (each ? (n / tile + 1 + count) * sizeof(double) : 0);
}

int gc_grad_norm(const gc_grads *grads, uint32_t p, double *total, float *norm, float *each, void *workspace,
                 gc_stream_t stream)
{
    const char *what = "gc_grad_norm";
    int rc;
    if ((rc = check_grads(grads, what)) || (rc = check_p(p, what)))
        return rc;
    if ((rc = check_workspace(grads, each != nullptr, workspace, what)))
        return rc;
    const Side side[] = {{"total", total, 8, true}, {"norm", norm, 4, true}, {"each", each, 4 * grads->count, true},
                         workspace_side(grads, each != nullptr, workspace)};
    if ((rc = check_sides(side, grads, nullptr, what)))
        return rc;
    hipStream_t st = as_stream(stream);
    if (each)
        launch_norm<true, false>(grads, p, ~0ull, workspace, total, norm, each, st);
    else
        launch_norm<false, false>(grads, p, ~0ull, workspace, total, norm, each, st);
    const uint32_t tile = norm_tile(grads, each != nullptr);
    const unsigned parts = norm_grid(grads->n, grads->count, tile, each != nullptr);
    if (!one_block(grads->n, grads->count, each != nullptr)) {
        const char *w = static_cast<const char *>(workspace);
        const dim3 grid(1 + (each ? (unsigned)grads->count : 0u));
        with_p(p, [&](auto P) {
            hipLaunchKernelGGL(k_grad_finish<P()>, grid, dim3(each ? kNormThreads : 64), 0, st, arg_of(grads), tile,
                               reinterpret_cast<const double *>(w), parts, reinterpret_cast<const double *>(w + kWsSlots),
                               total, norm, each);
        });
    }
    return launch_status(what);
}

int gc_grad_norm_root(const double *total, uint32_t p, float *norm, gc_stream_t stream)
{
    const char *what = "gc_grad_norm_root";
    int rc;
    if ((rc = check_p(p, what)))
        return rc;
    GC_REQUIRE(total && norm, "%s: null pointer", what);
    with_p(p, [&](auto P) {
        hipLaunchKernelGGL(k_grad_finish<P()>, dim3(1), dim3(64), 0, as_stream(stream), GradArg{nullptr, 0}, kTile,
                           total, 1u, nullptr, nullptr, norm, nullptr);
    });
    return launch_status(what);
}

int gc_grad_clip(const gc_grads *src, const gc_grads *dst, uint32_t p, double max_norm, const double *total,
                 float *norm, void *workspace, gc_stream_t stream)
{
    const char *what = "gc_grad_clip";
    int rc;
    if ((rc = check_grads(src, what)) || (rc = check_grads(dst, what)) || (rc = check_output(dst, what)) ||
        (rc = check_p(p, what)) || (rc = check_max_norm(max_norm, what)))
        return rc;
    GC_REQUIRE(src->count == dst->count, "%s: %llu tensors into %llu", what, (unsigned long long)src->count,
               (unsigned long long)dst->count);
    bool same = true;
    for (uint64_t s = 0; s <= src->count; ++s) {
        GC_REQUIRE(src->host_rec[2 * s + 1] == dst->host_rec[2 * s + 1],
                   "%s: the two lists differ in tensor sizes", what);
        same &= src->host_rec[2 * s] == dst->host_rec[2 * s];
    }
    if (!same && (rc = check_apart(src, dst, what)))
        return rc;
    if (!total && (rc = check_workspace(src, false, workspace, what)))
        return rc;
    const Side side[] = {{"norm", norm, 4, true}, {"total", total, 8, false},
                         workspace_side(src, false, total ? nullptr : workspace)};
    if ((rc = check_sides(side, src, dst, what)))
        return rc;
    hipStream_t st = as_stream(stream);
    const uint32_t tile = tile_of(src->n, src->count, kTile);
    if (!total && one_block(src->n, src->count)) {
        with_p(p, [&](auto P) {
            hipLaunchKernelGGL((k_grad_clip_one<P(), false>), dim3(1), dim3(kNormThreads), 0, st, arg_of(src),
                               arg_of(dst), nullptr, src->n, tile, max_norm, same, norm, nullptr);
        });
        return launch_status(what);
    }
    if (!total)
        launch_norm<false, false>(src, p, cold_elems(src), workspace, nullptr, nullptr, nullptr, st);
    const double *part = total ? total : static_cast<const double *>(workspace);
    const unsigned parts = total ? 1u : norm_grid(src->n, src->count, norm_tile(src));
    const uint64_t tiles = (src->n + tile - 1) / tile;
    const unsigned threads = scale_threads(tiles), grid = grid_of(tiles, threads, kScaleGrid);
    const GradArg a = arg_of(src), b = arg_of(dst);
    if (src->count <= kLdsRecs)
        hipLaunchKernelGGL((k_grad_scale<false, true>), dim3(grid), dim3(threads), 0, st, a, b, nullptr, src->n, tile,
                           cold_elems(src), (int)p, max_norm, part, parts, nullptr, same, norm, nullptr);
    else
        hipLaunchKernelGGL((k_grad_scale<false, false>), dim3(grid), dim3(threads), 0, st, a, b, nullptr, src->n, tile,
                           cold_elems(src), (int)p, max_norm, part, parts, nullptr, same, norm, nullptr);
    return launch_status(what);
}

int gc_grad_flatten_clip(const gc_grads *src, float *flat, uint32_t p, double max_norm, float *peak, float *norm,
                         void *workspace, gc_stream_t stream)
{
    const char *what = "gc_grad_flatten_clip";
    int rc;
    if ((rc = check_grads(src, what)) || (rc = check_p(p, what)) || (rc = check_max_norm(max_norm, what)))
        return rc;
    GC_REQUIRE(peak && (src->n == 0 || flat) && (reinterpret_cast<uintptr_t>(flat) & 3u) == 0,
               "%s: null or misaligned output", what);
    if ((rc = check_workspace(src, false, workspace, what)))
        return rc;
    const Side side[] = {{"the flat bucket", flat, 4 * src->n, true}, {"peak", peak, 4, true}, {"norm", norm, 4, true},
                         workspace_side(src, false, workspace)};
    if ((rc = check_sides(side, src, nullptr, what)))
        return rc;
    hipStream_t st = as_stream(stream);
    const uint32_t tile = tile_of(src->n, src->count, kTile);
    if (one_block(src->n, src->count)) {
        with_p(p, [&](auto P) {
            hipLaunchKernelGGL((k_grad_clip_one<P(), true>), dim3(1), dim3(kNormThreads), 0, st, arg_of(src),
                               GradArg{}, flat, src->n, tile, max_norm, false, norm, peak);
        });
        return launch_status(what);
    }
    launch_norm<false, true>(src, p, cold_elems(src), workspace, nullptr, nullptr, nullptr, st);
    const char *w = static_cast<const char *>(workspace);
    const uint64_t tiles = (src->n + tile - 1) / tile;
    const unsigned threads = scale_threads(tiles), grid = grid_of(tiles, threads, kScaleGrid);
    const unsigned parts = norm_grid(src->n, src->count, norm_tile(src));
    const GradArg a = arg_of(src);
    const double *part = reinterpret_cast<const double *>(w);
    const uint32_t *peaks = reinterpret_cast<const uint32_t *>(w + kWsPeak);
    if (src->count <= kLdsRecs)
        hipLaunchKernelGGL((k_grad_scale<true, true>), dim3(grid), dim3(threads), 0, st, a, GradArg{}, flat, src->n, tile,
                           cold_elems(src), (int)p, max_norm, part, parts, peaks, false, norm, peak);
    else
        hipLaunchKernelGGL((k_grad_scale<true, false>), dim3(grid), dim3(threads), 0, st, a, GradArg{}, flat, src->n,
                           tile, cold_elems(src), (int)p, max_norm, part, parts, peaks, false, norm, peak);
    return launch_status(what);
}

int gc_qsgd_decode_clip(const uint32_t *words, uint64_t n, const float *norm, uint32_t bits, const gc_lanes *lanes,
                        float alpha, const gc_grads *dst, uint32_t p, double max_norm, float *total_norm,
                        void *workspace, gc_stream_t stream)
{
    const char *what = "gc_qsgd_decode_clip";
    int rc;
    if ((rc = check_bits(bits, what)) || (rc = check_lanes(lanes, n, what)) || (rc = check_grads(dst, what)) ||
        (rc = check_output(dst, what)) || (rc = check_p(p, what)) || (rc = check_max_norm(max_norm, what)))
        return rc;
    const uint32_t s = (1u << bits) - 1u;
    GC_REQUIRE(lanes->offset == s && lanes->range == 2ull * s, "%s: lanes not made by gc_qsgd_layout", what);
    GC_REQUIRE(dst->n == n, "%s: the tensors hold %llu elements, the words %llu", what, (unsigned long long)dst->n,
               (unsigned long long)n);
    GC_REQUIRE(norm && total_norm && (n == 0 || words), "%s: null pointer", what);
    GC_REQUIRE(aligned16(words), "%s: words must be 16-byte aligned", what);
    if ((rc = check_workspace(dst, false, workspace, what)))
        return rc;
    const Side side[] = {{"the words", words, 4 * lanes->plane_words, false}, {"norm", norm, 4, false},
                         {"total_norm", total_norm, 4, true}, workspace_side(dst, false, workspace)};
    if ((rc = check_sides(side, nullptr, dst, what)))
        return rc;
    hipStream_t st = as_stream(stream);
    const LaneArg a{words, n, lanes->plane_words, norm, (float)s, alpha, (int32_t)(lanes->world * s), lanes->bits,
                    lanes->per_word, lanes->world * s, cold_part(lanes->plane_words, 4 * lanes->plane_words),
                    split_of(decode_tiles(lanes->plane_words), lanes->per_word)};
    const uint64_t quads = lanes->plane_words >> 2;
    const unsigned parts = grid_of((quads + 63) / 64, kNormThreads, kLaneGrid);
    uint64_t *part = static_cast<uint64_t *>(workspace);
    const GradArg d = arg_of(dst);
    const dim3 grid(grid_of(decode_tiles(lanes->plane_words) * a.split, kScaleThreads, kDecodeGrid));
    with_p(p, [&](auto P) {
        if (one_block(n, dst->count)) {
            hipLaunchKernelGGL(k_decode_clip_one<P()>, dim3(1), dim3(kNormThreads), 0, st, a, d, max_norm, total_norm);
            return;
        }
        hipLaunchKernelGGL(k_lane_norm<P()>, dim3(parts), dim3(kNormThreads), 0, st, a, part);
        if (dst->count <= kLdsRecs)
            hipLaunchKernelGGL((k_decode_clip<P(), true>), grid, dim3(kScaleThreads), 0, st, a, d, max_norm, part, parts,
                               total_norm);
        else
            hipLaunchKernelGGL((k_decode_clip<P(), false>), grid, dim3(kScaleThreads), 0, st, a, d, max_norm, part, parts,
                               total_norm);
    });
    return launch_status(what);
}

}  // extern "C"
