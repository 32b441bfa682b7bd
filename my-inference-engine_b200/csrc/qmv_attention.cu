// sm_100a kernels of the attention of many sequences: rotary embedding and
// append to a paged key/value cache, and causal grouped-query attention over
// packed prompts or over the cache.
//
// For a token at position p of its sequence and query head a (key/value head
// h = a / group):
//   s_j = scale * q . k_j for j <= p,  w_j = exp(s_j - max s) / sum_j exp(s_j - max s),
//   out = sum_j w_j v_j.
// The softmax runs in base 2 (scale * log2 e folded into one factor) and
// online: a running maximum m, sum l and unnormalised output o are rescaled
// by 2^(m_old - m_new) when a later key raises the maximum.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "qmv_attention.h"
#include "qmv_internal.h"

namespace qmv {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

__device__ unsigned int g_attention_status;

__device__ __forceinline__ void report(unsigned int bit) { atomicOr(&g_attention_status, bit); }

// --------------------------------------------------------- element types

// 16 bytes of a row as floats, and back.
template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ void load(const float *p, float v[4])
    {
        const float4 x = *(const float4 *)p;
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
    static __device__ __forceinline__ void store(float *p, const float v[4]) { *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]); }
    static __device__ __forceinline__ float to_float(float x) { return x; }
    static __device__ __forceinline__ float from_float(float x) { return x; }
};
template <> struct Elem<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void load(const __half *p, float v[8])
    {
        const uint4 x = *(const uint4 *)p;
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
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float v[8])
    {
        const uint4 x = *(const uint4 *)p;
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

// The last s in [0, n) with start[s] <= row (0 when there is none), by the
// 32 lanes of a warp together: 32 splits a step.
__device__ __forceinline__ int find_sequence(const int *__restrict__ start, int n, int row)
{
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 31) / 32;
        const int s = lo + lane * step;
        const bool below = s < lo + len && __ldg(start + s) <= row;
        const unsigned m = __ballot_sync(kFull, below);
        const int k = m ? 31 - __clz(m) : 0;
        const int end = lo + len;
        lo += k * step;
        len = min(step, end - lo);
    }
    return lo;
}

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

// Reports metadata out of range (one CTA of a launch calls it).
__device__ void check_metadata(const int *__restrict__ start, const int *__restrict__ length, int n, int tokens, int max_keys)
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
    if (bad) report(kStatusBadMetadata);
}

// ------------------------------------------------------ rope and append
//
// One CTA a token.  Its angles are formed once, in fixed point: position *
// base^(-2i / D) / 2 pi turns, the factor held as 64 bits of a turn, so the
// product modulo one turn is exact to position * 2^-65 turns and no position
// is too far for the f32 sine.  Threads then take 16-byte pieces of the
// first half of a head together with the pieces of the second half that they
// turn with, for all query and key heads, and the value pieces.
// Bound by bytes: q, k and v are read once and written once.

constexpr int kAppendThreads = 256;

struct Turns {
    unsigned long long f[64];  // fraction of a turn a position, times 2^64
};

template <typename T, typename KT, int D>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(AppendArgs a, const __grid_constant__ Turns turns)
{
    constexpr int V = Elem<T>::kVec, H = D / 2, U = H / V;  // pieces of a half head
    __shared__ float cs[H], sn[H];
    const int row = blockIdx.x;
    if (row == 0) check_metadata(a.start, a.length, a.sequences, a.tokens, max_keys_of(a.kv));
    const int s = find_sequence(a.start, a.sequences, row);
    const Seq sq = load_sequence(a.start, a.length, s, a.tokens, max_keys_of(a.kv));
    const int i = row - sq.row0, pos = sq.keys - sq.n + i;
    if (i < 0 || i >= sq.n || pos < 0) return;  // the same for the whole CTA
    const int page = __ldg(a.kv.table + (int64_t)s * a.kv.max_pages + (pos >> a.kv.page_shift));
    const bool stored = page >= 0 && page < a.kv.page_count;
    if (!stored && threadIdx.x == 0) report(kStatusBadMetadata);
    const bool rope = a.rope_base > 0.f;
    if (rope) {
        for (int e = threadIdx.x; e < H; e += kAppendThreads) {
            // the signed fraction of a turn in [-1/2, 1/2): angle / pi = 2 * fraction
            const long long frac = (long long)((unsigned long long)pos * turns.f[e]);
            sincospif((float)frac * 1.0842021724855044e-19f, &sn[e], &cs[e]);  // 2^-63
        }
        __syncthreads();
    }
    const int64_t slot = (int64_t)page * a.kv.page + (int64_t)(pos & ((1 << a.kv.page_shift) - 1)) * a.kv.k_pos;
    KT *kc = (KT *)const_cast<void *>(a.kv.k) + slot, *vc = (KT *)const_cast<void *>(a.kv.v) + slot;
    const T *q = (const T *)a.q + (int64_t)row * a.q_ld, *k = (const T *)a.k + (int64_t)row * a.k_ld;
    const T *v = (const T *)a.v + (int64_t)row * a.v_ld;
    T *qo = (T *)a.q_out + (int64_t)row * a.q_out_ld, *ko = (T *)a.k_out + (int64_t)row * a.k_out_ld;
    const int nq = a.q_out ? a.heads * U : 0, nk = a.kv_heads * U, total = nq + 2 * nk;
    for (int u = threadIdx.x; u < total; u += kAppendThreads) {
        const bool is_q = u < nq, is_v = u >= nq + nk;
        const int w = is_q ? u : is_v ? u - nq - nk : u - nq;
        const int head = w / U, e = (w % U) * V;
        const T *src = (is_q ? q : is_v ? v : k) + head * D + e;
        float x[V], y[V];
        Elem<T>::load(src, x);
        Elem<T>::load(src + H, y);
        if (rope && !is_v) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float c = cs[e + j], n = sn[e + j], xr = x[j] * c - y[j] * n, yr = x[j] * n + y[j] * c;
                x[j] = xr;
                y[j] = yr;
            }
        }
        T *out = is_q ? qo + head * D + e : ko + head * D + e;
        if (is_q || (!is_v && a.k_out)) {
            Elem<T>::store(out, x);
            Elem<T>::store(out + H, y);
        }
        if (!is_q && stored) {
            KT *dst = (is_v ? vc : kc) + head * a.kv.head + e;
            if constexpr (sizeof(T) == sizeof(KT)) {
                Elem<KT>::store(dst, x);
                Elem<KT>::store(dst + H, y);
            } else {
                __half2 p[4] = {__floats2half2_rn(x[0], x[1]), __floats2half2_rn(x[2], x[3]), __floats2half2_rn(y[0], y[1]),
                                __floats2half2_rn(y[2], y[3])};
                *(uint2 *)dst = *(const uint2 *)&p[0];
                *(uint2 *)(dst + H) = *(const uint2 *)&p[2];
            }
        }
    }
}

// ------------------------------------------------------ attention by rows
//
// One warp computes one (token, query head) in f32 on the CUDA cores: a lane
// a key for the scores, a lane D / 32 elements for the output.  Masked keys
// are never read.

template <typename T, typename KT, int D>
__device__ void attention_row(const AttnArgs &a, int row, int head, int s, const Seq &sq, float *qs)
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
    for (int j0 = 0; j0 < n_keys; j0 += 32) {
        const int j = j0 + lane;
        bool live = j < n_keys;
        int64_t ko = 0, vo = 0;
        if (live) {
            if (a.kv.table) {
                const int page = __ldg(a.kv.table + (int64_t)s * a.kv.max_pages + (j >> a.kv.page_shift));
                if (page < 0 || page >= a.kv.page_count) {
                    report(kStatusBadMetadata);
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
                Elem<KT>::load(k + e, x);
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
        for (int t = 0; t < 32; ++t) {
            if (!(alive >> t & 1u)) continue;
            const float pt = __shfl_sync(kFull, p, t);
            const int64_t at = __shfl_sync(kFull, vo, t);
            const KT *v = (const KT *)a.kv.v + at;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(pt, Elem<KT>::to_float(v[e * 32 + lane]), o[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e * 32 + lane] = Elem<T>::from_float(o[e] / l);
}

constexpr int kRowWarps = 4;

template <typename T, typename KT, int D>
__global__ void __launch_bounds__(kRowWarps * 32) attention_rows_kernel(AttnArgs a)
{
    __shared__ float qs[kRowWarps][D];
    if (blockIdx.x == 0 && blockIdx.y == 0) check_metadata(a.start, a.length, a.sequences, a.tokens, max_keys_of(a.kv));
    const int row = blockIdx.x, warp = threadIdx.x >> 5, head = blockIdx.y * kRowWarps + warp;
    const int s = find_sequence(a.start, a.sequences, row);
    const Seq sq = load_sequence(a.start, a.length, s, a.tokens, max_keys_of(a.kv));
    if (row < sq.row0 || row >= sq.row0 + sq.n || head >= a.heads) return;
    attention_row<T, KT, D>(a, row, head, s, sq, qs[warp]);
}

// The factors of `base` for head dimension d, to 64 bits of a turn; kept per
// calling thread for the last (base, d), since powl takes microseconds.
const Turns &turns_of(float base, int d)
{
    static thread_local Turns t{};
    static thread_local float have_base = 0.f;
    static thread_local int have_d = 0;
    if (base > 0.f && (base != have_base || d != have_d)) {
        const long double inv_2pi = 0.15915494309189533576888376337251436203445964574046L;
        for (int i = 0; i < d / 2; ++i) {
            long double f = powl((long double)base, -2.0L * i / d) * inv_2pi;
            f -= floorl(f);
            t.f[i] = (unsigned long long)(f * 18446744073709551616.0L);
        }
        have_base = base;
        have_d = d;
    }
    return t;
}

template <typename F> cudaError_t by_type(uint32_t type, uint32_t kv_type, int d, const F &f)
{
    if (type == kTypeF32 && kv_type == kTypeF32)
        return d == 64 ? f(float{}, float{}, std::integral_constant<int, 64>{}) : f(float{}, float{}, std::integral_constant<int, 128>{});
    if (type == kTypeF32 && kv_type == kTypeF16)
        return d == 64 ? f(float{}, __half{}, std::integral_constant<int, 64>{}) : f(float{}, __half{}, std::integral_constant<int, 128>{});
    if (type == kTypeF16 && kv_type == kTypeF16)
        return d == 64 ? f(__half{}, __half{}, std::integral_constant<int, 64>{}) : f(__half{}, __half{}, std::integral_constant<int, 128>{});
    if (type == kTypeBF16 && kv_type == kTypeBF16)
        return d == 64 ? f(__nv_bfloat16{}, __nv_bfloat16{}, std::integral_constant<int, 64>{})
                       : f(__nv_bfloat16{}, __nv_bfloat16{}, std::integral_constant<int, 128>{});
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_paged_append(const AppendArgs &a, cudaStream_t s)
{
    const Turns &turns = turns_of(a.rope_base, a.head_dim);
    return by_type(a.type, a.kv_type, a.head_dim, [&](auto t, auto kt, auto d) {
        paged_append_kernel<decltype(t), decltype(kt), d.value><<<(unsigned)a.tokens, kAppendThreads, 0, s>>>(a, turns);
        return cudaGetLastError();
    });
}

cudaError_t launch_attention_rows(const AttnArgs &a, cudaStream_t s)
{
    return by_type(a.type, a.kv_type, a.head_dim, [&](auto t, auto kt, auto d) {
        const dim3 grid((unsigned)a.tokens, (unsigned)((a.heads + kRowWarps - 1) / kRowWarps));
        attention_rows_kernel<decltype(t), decltype(kt), d.value><<<grid, kRowWarps * 32, 0, s>>>(a);
        return cudaGetLastError();
    });
}

cudaError_t attention_status(unsigned int *out, bool clear)
{
    cudaError_t e = cudaMemcpyFromSymbol(out, g_attention_status, sizeof(unsigned int));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0u;
        e = cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(unsigned int));
    }
    return e;
}

}  // namespace qmv
