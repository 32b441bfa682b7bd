// Device code shared by the attention kernels: element types, the metadata of
// a ragged batch, and one row computed plainly.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "qmv_attention.h"

namespace qmv {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void report(unsigned int *status, unsigned int bit) { atomicOr(status, bit); }

// 2^x (2 ulp; results below 2^-126 become 0).
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two floats rounded to KT in one word, a in the low half.
template <typename KT> __device__ __forceinline__ uint32_t pack2(float a, float b)
{
    uint32_t w;
    if constexpr (std::is_same<KT, __half>::value)
        *(__half2 *)&w = __floats2half2_rn(a, b);
    else
        *(__nv_bfloat162 *)&w = __floats2bfloat162_rn(a, b);
    return w;
}

// The power of two that brings a row's largest |x| into [2^14, 2^15): any but
// those of rows below 2^-100, whose product with the scale has to stay normal.
constexpr int kUnitMin = -113, kUnitMax = 114;

// What is left of (a, b) after their f16 rounding, as f16.
__device__ __forceinline__ uint32_t pack2_rest(float a, float b, uint32_t hi)
{
    const float2 h = __half22float2(*(const __half2 *)&hi);
    return pack2<__half>(a - h.x, b - h.y);
}

// --------------------------------------------------------- element types

// 16 bytes of a row as floats, and back.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ void unpack(const uint4 &x, float v[4])
    {
        v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
    }
    static __device__ __forceinline__ void store(float *p, const float v[4]) { *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]); }
    static __device__ __forceinline__ float to_float(float x) { return x; }
    static __device__ __forceinline__ float from_float(float x) { return x; }
};
template <> struct Elem<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void unpack(const uint4 &x, float v[8])
    {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*(const __half2 *)&w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(__half *p, const float v[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) *(__half2 *)&w[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void unpack(const uint4 &x, float v[8])
    {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float v[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) *(__nv_bfloat162 *)&w[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
};

// ------------------------------------------------------------ metadata

struct Seq {
    int row0;  // first row
    int n;     // new tokens (0: left out)
    int keys;  // cached positions, new tokens included
};

__device__ __forceinline__ Seq load_sequence(const int *__restrict__ start, const int *__restrict__ length, int s,
                                             int tokens, int max_keys)
{
    const int a = __ldg(start + s), b = __ldg(start + s + 1);
    Seq q{a, b - a, b - a};
    bool ok = a >= 0 && a <= b && b <= tokens;
    if (length != nullptr) {
        q.keys = __ldg(length + s);
        ok = ok && q.keys >= 0 && q.keys <= max_keys;
    }
    if (!ok) q.n = q.keys = 0;
    return q;
}

__device__ __forceinline__ int max_keys_of(const KvView &kv) { return kv.table ? kv.max_pages << kv.page_shift : 0x7fffffff; }

// The sequence that owns a row (the last s with start[s] <= row; 0 when there
// is none) by the 32 lanes of a warp together: 32 splits a step, and the last
// step's lanes bring the candidates' metadata along.
__device__ __forceinline__ int find_sequence(const int *__restrict__ start, const int *__restrict__ length, int n, int row, int tokens, int max_keys,
                                             Seq *found)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (len > 32) {
        const int step = (len + 31) / 32, s = lo + lane * step, end = lo + len;
        const unsigned m = __ballot_sync(kFull, s < end && __ldg(start + s) <= row);
        lo += (m ? 31 - __clz(m) : 0) * step;
        len = min(step, end - lo);
    }
    Seq q{0x7fffffff, 0, 0};
    if (lane < len) q = load_sequence(start, length, lo + lane, tokens, max_keys);
    const unsigned m = __ballot_sync(kFull, lane < len && q.row0 <= row);
    const int k = m ? 31 - __clz(m) : 0;
    *found = Seq{__shfl_sync(kFull, q.row0, k), __shfl_sync(kFull, q.n, k), __shfl_sync(kFull, q.keys, k)};
    return lo + k;
}

// Reports metadata out of range (one CTA of a launch calls it).
__device__ __forceinline__ void check_metadata(unsigned int *status, const int *__restrict__ start, const int *__restrict__ length, int n, int tokens, int max_keys)
{
    bool bad = false;
    for (int s = threadIdx.x; s < n; s += blockDim.x) {
        const int a = __ldg(start + s), b = __ldg(start + s + 1);
        bad |= !(a >= 0 && a <= b && b <= tokens);
        if (length != nullptr) {
            const int k = __ldg(length + s);
            bad |= k < 0 || k > max_keys;
        }
    }
    if (bad) report(status, kStatusBadMetadata);
}

// ------------------------------------------------------ shares of the work
//
// A launch's work is a line of places, dealt to its CTAs in equal shares in
// order.  Where a share's border falls inside an item, the share that holds
// the item's beginning joins it: the others leave what they have (maximum, sum,
// unnormalised output) in scratch and set a flag; it ends its own part last, so
// as a rule it finds them there, adds them in order and writes the output.
// CTA b has share gridDim.x - 1 - b: a share waits only for later shares,
// whose CTAs were dispatched before its own, so every wait ends however
// many CTAs are resident.  (The hardware dispatches CTAs in the order of their
// index; CUDA does not promise it, and where it did not hold a wait could run
// into its limit, which the status reports.  A second kernel for the join took
// 4 to 10 us.)
//
// Flags carry a number of the launch's own, so scratch needs no clearing.  A
// captured launch has a count beside it (LaunchTag), so that each replay has its
// own number too, and a flag that a share set after its wait had expired is
// nothing to the next replay.

// Division by a number the host knows: its floor(2^64 / d) + 1 (exact for
// dividends below 2^31; within 1 above, and corrected).
struct Divisor {
    unsigned long long magic;
    int d;
};

inline Divisor divisor(int d) { return Divisor{d > 1 ? ~0ull / (unsigned long long)d + 1 : ~0ull, d}; }

struct Deal {
    long long each;
    int more, shares;  // the first `more` shares get one place more
    // No share below `least` places (but the only one): a join costs more than a
    // short share saves.
    static __device__ __forceinline__ Deal of(long long total, const Divisor &d, int least)
    {
        Deal t;
        if (total >= (long long)least * d.d) {
            t.each = (long long)__umul64hi((unsigned long long)total, d.magic);
            if (t.each * d.d > total) --t.each;
            t.shares = d.d;
        } else {
            t.shares = max(1, (int)total / least);
            t.each = (int)total / t.shares;
        }
        t.more = (int)(total - t.each * t.shares);
        return t;
    }
    __device__ __forceinline__ long long first(int c) const { return each * c + (c < more ? c : more); }
    // The share that place u falls to: an estimate, then exactly.
    __device__ __forceinline__ int holder(long long u) const
    {
        int c = min(shares - 1, (int)((float)u / ((float)each + (float)more / (float)shares)));
        while (first(c) > u) --c;
        while (c + 1 < shares && first(c + 1) <= u) ++c;
        return c;
    }
};

__device__ __forceinline__ int my_share() { return (int)(gridDim.x - 1 - blockIdx.x); }

constexpr unsigned long long kWaitLimitNs = 2000000000ull;

__device__ __forceinline__ unsigned long long now_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void flag_set(unsigned long long *flag, unsigned long long launch)
{
    __threadfence();
    asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(flag), "l"(launch) : "memory");
}

// Waits (bounded) for a flag; false when the wait expired.
__device__ __forceinline__ bool flag_wait(const unsigned long long *flag, unsigned long long launch, unsigned long long limit_ns = kWaitLimitNs)
{
    unsigned long long v, t0 = 0;
    for (uint32_t n = 0;; ++n) {
        asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(flag) : "memory");
        if (v == launch) return true;
        if (n == 0) t0 = now_ns();
        if ((n & 63u) == 63u && now_ns() - t0 > limit_ns) return false;
    }
}

// The number of this launch, by one thread of every CTA, once.  All CTAs of a
// replay count, and each before it knows the number, so the count is between
// k gridDim.x and (k + 1) gridDim.x - 1 for all of replay k.
__device__ __forceinline__ unsigned long long number_of(const LaunchTag &tag)
{
    return tag.number + (tag.count ? atomicAdd(tag.count, 1ull) / gridDim.x : 0ull);
}

// Sum over the CTA's NT threads of one value each, and the exclusive prefix.
template <int NT> __device__ __forceinline__ long long block_scan(long long v, long long *total)
{
    __shared__ long long scratch[NT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(kFull, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += scratch[w];
        all += scratch[w];
    }
    *total = all;
    return before + x - v;
}

// Where this CTA's share begins: Iter at its first unit, places [u0, u1), by
// all threads of the CTA together.  A thread sums the cost of a run of
// sequences, and the one whose run holds the place walks to it.
template <typename Iter> struct Start {
    Iter it;  // it.s == sequences: nothing
    long long u0, u1;
    Deal deal;
};

template <int NT, typename Plan, typename Iter> __device__ __forceinline__ void find_start(const Plan &p, Start<Iter> *out)
{
    const int per = p.sequences <= NT ? 1 : (p.sequences + NT - 1) / NT, s0 = min((int)threadIdx.x * per, p.sequences), s1 = min(s0 + per, p.sequences);
    long long v = 0, all;
    Seq q{0, 0, 0};
    for (int s = s0; s < s1; ++s) {
        q = p.seq(s);
        v += p.cost(q);
    }
    long long at = block_scan<NT>(v, &all);
    const Deal deal = Deal::of(all, p.ctas, Plan::kLeast);
    const int c = my_share();
    const long long u0 = deal.first(c), u1 = deal.first(c + 1);
    if (c >= deal.shares || u0 >= u1) {
        if (threadIdx.x == 0) {
            out->it.s = p.sequences;
            out->u0 = out->u1 = 0;
        }
    } else if (u0 >= at && u0 < at + v) {
        int s = s0;
        if (per > 1)
            for (long long cost; u0 >= at + (cost = p.cost(q = p.seq(s))); ++s) at += cost;
        Iter it;
        it.begin(p, s, q, u0 - at, u0);
        out->it = it;
        out->u0 = u0;
        out->u1 = u1;
        out->deal = deal;
    }
    __syncthreads();
}

// ------------------------------------------------------ attention by rows
//
// One warp computes one (token, query head) in f32 on the CUDA cores: a lane
// a key for the scores, a lane D / 32 elements for the output.  Masked keys are
// never read.  The faster kernels come back to it for rows that are not finite:
// a masked key's weight of 0 times a NaN or infinite value must not reach a
// sum, and theirs does.

template <typename T, typename KT, int D>
__device__ __noinline__ void attention_row(const AttnArgs &a, int row, int head, int s, const Seq &sq, float *qs)
{
    constexpr int V = Elem<KT>::kVec, E = D / 32;
    const int lane = threadIdx.x & 31, h = head / a.group;
    const int n_keys = sq.keys - sq.n + (row - sq.row0) + 1;
    T *out = (T *)a.out + (int64_t)row * a.out_ld + head * D;
    if (n_keys <= 0) {
        for (int e = lane; e < D; e += 32) out[e] = Elem<T>::from_float(0.f);
        return;
    }
    const T *q = (const T *)a.q + (int64_t)row * a.q_ld + head * D;
    __syncwarp();
    for (int e = lane; e < D; e += 32) qs[e] = Elem<T>::to_float(q[e]);
    __syncwarp();
    const float f = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    // From the last key back, as far as the row is not NaN all over: rows at and
    // behind a NaN token mostly have a NaN key and value of their own.  A prompt
    // of 8192 NaN tokens (bf16, 28/4/128) takes 6.7 ms, from the first key 324.
    bool lost = false;
    for (int j1 = n_keys; j1 > 0 && !lost; j1 -= 32) {
        const int j = j1 - 32 + lane;
        bool live = j >= 0;
        int64_t ko = 0, vo = 0;
        if (live) {
            if (a.kv.table) {
                const int page = __ldg(a.kv.table + (int64_t)s * a.kv.max_pages + (j >> a.kv.page_shift));
                if (page < 0 || page >= a.kv.page_count) {
                    report(a.status, kStatusBadMetadata);
                    live = false;
                } else {
                    ko = (int64_t)page * a.kv.page + (int64_t)(j & ((1 << a.kv.page_shift) - 1)) * a.kv.k_pos;
                    vo = ko;
                }
            } else {
                ko = (int64_t)(sq.row0 + j) * a.kv.k_pos;
                vo = (int64_t)(sq.row0 + j) * a.kv.v_pos;
            }
            ko += h * a.kv.head;
            vo += h * a.kv.head;
        }
        float sc = -INFINITY;
        if (live) {
            const KT *k = (const KT *)a.kv.k + ko;
            float acc = 0.f;
            for (int e = 0; e < D; e += V) {
                float x[V];
                Elem<KT>::unpack(*(const uint4 *)(k + e), x);
#pragma unroll
                for (int t = 0; t < V; ++t) acc = fmaf(x[t], qs[e + t], acc);
            }
            sc = acc * f;
        }
        float mt = sc;
        bool nan = isnan(sc);
#pragma unroll
        for (int d = 16; d; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(kFull, mt, d));
        if (__any_sync(kFull, nan)) mt = NAN;
        const float mn = isnan(mt) || isnan(m) ? NAN : fmaxf(m, mt);
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float p = live ? exp2f(sc - ms) : 0.f;
        const float fix = m == -INFINITY ? 0.f : exp2f(m - ms);
        m = mn;
        float sum = p;
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
        l = l * fix + sum;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= fix;
        const unsigned alive = __ballot_sync(kFull, live);
#pragma unroll 8
        for (int t = 0; t < 32; ++t) {
            const float pt = __shfl_sync(kFull, p, t);
            const int64_t at = __shfl_sync(kFull, vo, t);
            if (!(alive >> t & 1u)) continue;
            const KT *v = (const KT *)a.kv.v + at;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(pt, Elem<KT>::to_float(v[e * 32 + lane]), o[e]);
        }
        bool all_nan = true;  // and so they stay
#pragma unroll
        for (int e = 0; e < E; ++e) all_nan &= isnan(o[e]);
        lost = __all_sync(kFull, all_nan);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e * 32 + lane] = Elem<T>::from_float(o[e] / l);
}

}  // namespace

}  // namespace qmv
