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
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "qmv_attention.cuh"
#include "qmv_internal.h"

namespace qmv {

namespace {

__device__ unsigned int g_attention_status;
__device__ unsigned long long g_launch_count[kLaunchCounts];

// ------------------------------------------------------ rope and append
//
// One CTA a token, or two neighbours where there are many, so that the chain
// from the sequence over its length and page to the first store is paid once
// for both.  Each token's angles are formed once, in fixed point: position *
// base^(-2i / D) / 2 pi turns, the factor held as 64 bits of a turn, so the
// product modulo one turn is exact to position * 2^-63 turns (the factor is cut,
// after powl and the product) and no position is too far for the f32 sine.  Threads then take 16-byte pieces of the
// first half of a head together with the pieces of the second half that they
// turn with, for all query and key heads, and the value pieces; a thread's
// first piece is on its way while the sequence, the page and the angles are found.
// Bound by bytes, q, k and v being read once and written once, and below some
// thousand tokens by that chain: 6789 tokens (bf16, 28/4/128; 125 MB) take 26 us,
// 4.8 TB/s, 20000 5.5 TB/s.  With four or eight tokens a CTA registers cost more
// than the chain saves.

constexpr int kAppendThreads = 512;  // at most: a thread a piece, as far as they go

struct Turns {
    unsigned long long f[64];  // fraction of a turn a position, times 2^64
};

template <typename T, typename KT, int D, int R>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(AppendArgs a, const __grid_constant__ Turns turns)
{
    constexpr int V = Elem<T>::kVec, H = D / 2, U = H / V;  // pieces of a half head
    __shared__ float cs[R][H], sn[R][H];
    __shared__ int position[R];  // -1: not a token to append
    __shared__ int64_t slot[R];  // its place in a page's keys, -1: nowhere
    const int row0 = (int)blockIdx.x * R, warp = threadIdx.x >> 5;
    const int nq = a.q_out ? a.heads * U : 0, nk = a.kv_heads * U, total = nq + 2 * nk;
    uint4 raw_x[R], raw_y[R];
    auto fetch = [&](int i, int u) {
        const int row = row0 + i;
        if (row >= a.tokens) return;
        const bool is_q = u < nq, is_v = u >= nq + nk;
        const int w = is_q ? u : is_v ? u - nq - nk : u - nq;
        const T *src = is_q ? (const T *)a.q + (int64_t)row * a.q_ld : is_v ? (const T *)a.v + (int64_t)row * a.v_ld : (const T *)a.k + (int64_t)row * a.k_ld;
        src += w / U * D + (w % U) * V;
        raw_x[i] = *(const uint4 *)src;
        raw_y[i] = *(const uint4 *)(src + H);
    };
    if ((int)threadIdx.x < total) {
#pragma unroll
        for (int i = 0; i < R; ++i) fetch(i, threadIdx.x);
    }
    if (row0 == 0) check_metadata(a.status, a.start, a.length, a.sequences, a.tokens, max_keys_of(a.kv));
    static_assert(R <= 2, "a warp a token, and two warps at least");
    int page = -1, pos = -1;  // of token `warp`
    if (warp < R) {
        const int row = row0 + warp;
        Seq sq;
        const int s = find_sequence(a.start, a.length, a.sequences, row, a.tokens, max_keys_of(a.kv), &sq);
        const int at = row - sq.row0;
        if (at >= 0 && at < sq.n) pos = sq.keys - sq.n + at;
        if (pos >= 0) page = __ldg(a.kv.table + (int64_t)s * a.kv.max_pages + (pos >> a.kv.page_shift));
        if ((threadIdx.x & 31) == 0) position[warp] = pos < 0 ? -1 : pos;
    }
    __syncthreads();
    const bool rope = a.rope_base > 0.f;
    if (rope) {  // while the pages' numbers are on their way
        for (int e = threadIdx.x; e < R * H; e += (int)blockDim.x) {
            // the signed fraction of a turn in [-1/2, 1/2): angle / pi = 2 * fraction
            const long long frac = (long long)((unsigned long long)position[e / H] * turns.f[e % H]);
            sincospif((float)frac * 1.0842021724855044e-19f, &sn[e / H][e % H], &cs[e / H][e % H]);  // 2^-63
        }
    }
    if (warp < R && (threadIdx.x & 31) == 0) {
        const bool stored = page >= 0 && page < a.kv.page_count;
        if (pos >= 0 && !stored) report(a.status, kStatusBadMetadata);
        slot[warp] = stored ? (int64_t)page * a.kv.page + (int64_t)(pos & ((1 << a.kv.page_shift) - 1)) * a.kv.k_pos : -1;
    }
    __syncthreads();
    for (int u = threadIdx.x; u < total; u += (int)blockDim.x) {
        const bool is_q = u < nq, is_v = u >= nq + nk;
        const int w = is_q ? u : is_v ? u - nq - nk : u - nq;
        const int head = w / U, e = (w % U) * V;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (position[i] < 0) continue;
            if (u != (int)threadIdx.x) fetch(i, u);
            float x[V], y[V];
            Elem<T>::unpack(raw_x[i], x);
            Elem<T>::unpack(raw_y[i], y);
            if (rope && !is_v) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float c = cs[i][e + j], n = sn[i][e + j], xr = x[j] * c - y[j] * n, yr = x[j] * n + y[j] * c;
                    x[j] = xr;
                    y[j] = yr;
                }
            }
            if (is_q || (!is_v && a.k_out)) {
                T *out = is_q ? (T *)a.q_out + (int64_t)(row0 + i) * a.q_out_ld : (T *)a.k_out + (int64_t)(row0 + i) * a.k_out_ld;
                out += head * D + e;
                Elem<T>::store(out, x);
                Elem<T>::store(out + H, y);
            }
            if (!is_q && slot[i] >= 0) {
                KT *dst = (KT *)const_cast<void *>(is_v ? a.kv.v : a.kv.k) + slot[i] + head * a.kv.head + e;
                if constexpr (sizeof(T) == sizeof(KT)) {
                    Elem<KT>::store(dst, x);
                    Elem<KT>::store(dst + H, y);
                } else {
                    *(uint2 *)dst = make_uint2(pack2<KT>(x[0], x[1]), pack2<KT>(x[2], x[3]));
                    *(uint2 *)(dst + H) = make_uint2(pack2<KT>(y[0], y[1]), pack2<KT>(y[2], y[3]));
                }
            }
        }
    }
}

// ------------------------------------------------- paged decode attention
//
// Few query rows over many cached keys: bound by the bytes of the cache, each
// read once for all the query heads of its key/value head.
//
// Rows r = token * group + head-in-group of one (sequence, key/value head)
// are cut into tiles of 16, the M of mma.sync m16n8k16; a row tile of one
// sequence and head is an item, its keys in blocks of 64 are its units, and
// all units of the launch, in order, are dealt evenly to the CTAs (two an
// SM, so that one streams while the other ends an item), and ragged lengths
// cost nothing.  Each of the 4 warps takes 16 keys of every unit, streams
// them through its own cp.async ring (the rings together keep 128 KB an SM in
// flight, with no barrier between warps) and holds its own running maximum,
// sum and output in registers; the warps meet once per item.
// tcgen05 is not used: its M of 64 or more would be mostly empty rows here,
// and the tensor work is a tenth of the time the bytes take.

constexpr int kDcWarps = 4;
constexpr int kDcPerSm = 2;
constexpr int kDcThreads = kDcWarps * 32;
constexpr int kDcKeys = 16;                   // keys of a warp's step
constexpr int kDcUnit = kDcKeys * kDcWarps;   // keys of a unit
constexpr int kDcRows = 16;                   // rows of a tile
// What an item costs beside its keys, in units: loading its queries, the
// warps' meeting and the output take 3700 cycles, a unit 1100 (D = 128).
// Dealt without it, 64 sequences of 16..8192 positions took 66 us instead of 39.
constexpr int kDcItemCost = 3;

template <int D> struct Dc {
    static constexpr uint32_t kRow = D * 2;                    // bytes of a key
    static constexpr uint32_t kStep = 2 * kDcKeys * kRow;      // K and V of a step
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kRing = kStep * kStages * kDcWarps;
    static constexpr uint32_t kMerge = kDcWarps * 8 * D * 4;   // 8 rows of every warp
    static constexpr uint32_t kSmem = kRing + kMerge + kDcWarps * kDcRows * 8;
    static constexpr int kPartial = kDcRows * D + 2 * kDcRows;  // floats: o, m, l
    // rows of D floats, 8-float blocks exchanged by the row so that the 8
    // rows a warp writes at once fall on different banks
    static __device__ __forceinline__ int at(int row, int col) { return row * D + (col ^ ((row & 7) * 8)); }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16u : 0u) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename KT> __device__ __forceinline__ void mma16816(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1)
{
    if constexpr (sizeof(KT) == 2 && std::is_same<KT, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a sequence costs, in blocks of keys: row tiles x heads items, each of
// its key blocks and of kDcItemCost for its beginning and end.
struct DcPlan {
    static constexpr int kLeast = 2;  // units: one takes as long, for its latencies
    const int *start, *length;
    int sequences, tokens, max_keys, kv_heads, group;
    Divisor ctas;
    __device__ __forceinline__ Seq seq(int s) const { return load_sequence(start, length, s, tokens, max_keys); }
    __device__ __forceinline__ int tiles(const Seq &q) const { return (q.n * group + kDcRows - 1) / kDcRows; }
    __device__ __forceinline__ int blocks(const Seq &q) const { return q.keys > 0 ? (q.keys + kDcUnit - 1) / kDcUnit : 1; }
    __device__ __forceinline__ long long cost(const Seq &q) const { return (long long)tiles(q) * kv_heads * (blocks(q) + kDcItemCost); }
};

// Walks units in order: sequence, head, row tile, key block.  A unit's place
// is its item's first place + kDcItemCost + blk; a CTA has the units whose
// places fall in its share.
struct DcIter {
    Seq q;
    int s, h, rt, blk, rts, blks;
    long long u;  // the unit's place
    __device__ __forceinline__ void enter(const DcPlan &p)
    {
        rts = blks = 0;
        while (s < p.sequences) {
            q = p.seq(s);
            rts = p.tiles(q);
            blks = p.blocks(q);
            if (rts > 0) break;
            ++s;
        }
    }
    // The first unit at or behind place rel of sequence s_ (one with tiles),
    // and its own place, where rel is place u0.
    __device__ __forceinline__ void begin(const DcPlan &p, int s_, const Seq &q_, long long rel, long long u0)
    {
        s = s_;
        q = q_;
        rts = p.tiles(q);
        blks = p.blocks(q);
        const int span = blks + kDcItemCost;
        int item = (int)((float)rel / (float)span);  // an estimate, then exactly
        while ((long long)item * span > rel) --item;
        while ((long long)(item + 1) * span <= rel) ++item;
        const int at = (int)(rel - (long long)item * span);
        blk = max(0, at - kDcItemCost);
        h = item / rts;
        rt = item - h * rts;
        u = u0 + kDcItemCost + blk - at;
    }
    __device__ __forceinline__ void next(const DcPlan &p)
    {
        ++u;
        if (++blk < blks) return;
        u += kDcItemCost;
        blk = 0;
        if (++rt < rts) return;
        rt = 0;
        if (++h < p.kv_heads) return;
        h = 0;
        ++s;
        enter(p);
    }
};

// Writes 4 columns of an output row; true when one is not finite.
template <typename T> __device__ __forceinline__ bool store4(T *out, const float4 &v)
{
    if constexpr (sizeof(T) == 4) {
        *(float4 *)out = v;
    } else {
        *(uint2 *)out = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
    }
    return !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
}

template <typename T, typename KT, int D>
__global__ void __launch_bounds__(kDcThreads, kDcPerSm) decode_attention_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ DcPlan plan,
                                                                                 float *partials, unsigned long long *flags, LaunchTag tag)
{
    using C = Dc<D>;
    constexpr int NQ = sizeof(T) == 4 ? 2 : 1;  // f16 pairs for f32 activations
    constexpr int KS = D / 16, NT = D / 8;
    // the weights' exponent offset: the reference is the maximum itself, so f16
    // weights may reach 2^15.875 (f16 ends at 2^16 - 32; a score so large that
    // its rounding passes that gives an infinity, and its row is computed again)
    // and stay normal down to 2^-29 of the largest (as pairs: 22 bits to 2^-18,
    // 2^-40 below)
    constexpr float kLift = std::is_same<KT, __half>::value ? 15.875f : 0.f;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ unsigned bad_rows;
    __shared__ Start<DcIter> begin;
    __shared__ unsigned long long number;
    float *merge = (float *)(smem + C::kRing);
    float2 *ml = (float2 *)(smem + C::kRing + C::kMerge);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3, grp = lane >> 2;
    if (blockIdx.x == 0) check_metadata(a.status, a.start, a.length, a.sequences, a.tokens, plan.max_keys);
    if (tid == 0) bad_rows = 0u;
    if (tid == kDcThreads - 1) number = number_of(tag);
    find_start<kDcThreads>(plan, &begin);
    const long long u1 = begin.u1;
    DcIter it = begin.it, pf = it;
    if (it.s >= plan.sequences || it.u >= u1) return;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (uint32_t)warp * C::kStep * C::kStages;
    const int mask = (1 << a.kv.page_shift) - 1;

    // the page of the next step to fetch, loaded one step ahead of its use
    auto page_of = [&](const DcIter &i) {
        const int j0 = i.blk * kDcUnit + warp * kDcKeys;
        return j0 < i.q.keys ? __ldg(a.kv.table + (int64_t)i.s * a.kv.max_pages + (j0 >> a.kv.page_shift)) : -1;
    };
    uint32_t to_stage = 0u;  // its stage
    int page = page_of(pf);
    auto issue = [&]() {
        if (pf.u < u1) {
            const int j0 = pf.blk * kDcUnit + warp * kDcKeys;
            if (j0 < pf.q.keys) {
                const bool good = page >= 0 && page < a.kv.page_count;
                if (!good && lane == 0) report(a.status, kStatusBadMetadata);
                const int64_t base = (int64_t)(good ? page : 0) * a.kv.page + (int64_t)(j0 & mask) * a.kv.k_pos + (int64_t)pf.h * a.kv.head;
                const KT *k = (const KT *)a.kv.k + base, *v = (const KT *)a.kv.v + base;
                const uint32_t dst = ring + to_stage * C::kStep;
                constexpr int CH = D / 8;  // 16-byte pieces of a key
                const int c = lane % CH;
#pragma unroll
                for (int r0 = 0; r0 < kDcKeys; r0 += 32 / CH) {
                    const int r = r0 + lane / CH;
                    const bool live = good && j0 + r < pf.q.keys;
                    const int64_t off = live ? (int64_t)r * a.kv.k_pos + c * 8 : 0;
                    const uint32_t to = dst + (uint32_t)r * C::kRow + (uint32_t)((c ^ (r & 7)) * 16);
                    cp16(to, k + off, live);
                    cp16(to + kDcKeys * C::kRow, v + off, live);
                }
            }
            to_stage = to_stage + 1 == C::kStages ? 0u : to_stage + 1;
            pf.next(plan);
            if (pf.u < u1) page = page_of(pf);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < C::kStages - 1; ++i) issue();

    uint32_t qf[NQ][KS][4];
    float o[NT][4], m[2], l[2], factor[2];
    int lim[2];
    uint32_t stage = 0u;
    bool fresh = true;  // at the first unit of a segment, this CTA's part of an item
    int first_blk = 0;  // its key block
    while (it.u < u1) {
        if (fresh) {
            fresh = false;
            first_blk = it.blk;
            // the item's query rows as A fragments: rows grp and grp + 8
            const int rows = it.q.n * a.group - it.rt * kDcRows;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = it.rt * kDcRows + grp + 8 * half, token = r / a.group;
                const bool live = grp + 8 * half < rows;
                lim[half] = live ? it.q.keys - it.q.n + token + 1 : 0;
                const T *q = (const T *)a.q + (int64_t)(it.q.row0 + (live ? token : 0)) * a.q_ld +
                             (int64_t)(it.h * a.group + (live ? r - token * a.group : 0)) * D;
                m[half] = -INFINITY;
                l[half] = 0.f;
                factor[half] = a.scale * kLog2e;
                if constexpr (NQ == 1) {
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        qf[0][k][half] = live ? *(const uint32_t *)(q + 16 * k + 2 * quad) : 0u;
                        qf[0][k][2 + half] = live ? *(const uint32_t *)(q + 16 * k + 8 + 2 * quad) : 0u;
                    }
                } else {
                    // x = (hi + lo) 2^-e with the row's largest |x| in
                    // [2^14, 2^15) after the shift: 22 bits a value
                    float2 x[KS][2];
                    float big = 0.f;
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            x[k][p] = live ? *(const float2 *)(q + 16 * k + 8 * p + 2 * quad) : make_float2(0.f, 0.f);
                            big = fmaxf(big, fmaxf(fabsf(x[k][p].x), fabsf(x[k][p].y)));
                        }
                    big = fmaxf(big, __shfl_xor_sync(kFull, big, 1));
                    big = fmaxf(big, __shfl_xor_sync(kFull, big, 2));
                    int e = 14 - (int)((__float_as_uint(big) >> 23) & 255u) + 127;
                    e = min(max(e, kUnitMin), kUnitMax);
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                    factor[half] *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            const float y0 = x[k][p].x * up, y1 = x[k][p].y * up;
                            const uint32_t hi = pack2<__half>(y0, y1);
                            qf[0][k][2 * p + half] = hi;
                            qf[NQ - 1][k][2 * p + half] = pack2_rest(y0, y1, hi);
                        }
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 2) : "memory");
        __syncwarp();
        issue();  // refills the stage read in the previous step
        const int j0 = it.blk * kDcUnit + warp * kDcKeys;
        if (j0 < it.q.keys) {
            const uint32_t ks = ring + stage * C::kStep, vs = ks + kDcKeys * C::kRow;
            float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            {
                const int r = (lane & 7) + ((lane >> 4) << 3), c0 = (lane >> 3) & 1;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    ldsm4(b, ks + (uint32_t)r * C::kRow + (uint32_t)(((2 * k + c0) ^ (r & 7)) * 16));
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        mma16816<KT>(sc[0], qf[n][k], b[0], b[1]);
                        mma16816<KT>(sc[1], qf[n][k], b[2], b[3]);
                    }
                }
            }
            float p[2][4];
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int half = e >> 1, j = j0 + 8 * t + 2 * quad + (e & 1);
                    p[t][e] = j < lim[half] ? sc[t][e] : -INFINITY;
                    top[half] = fmaxf(top[half], p[t][e]);
                }
            float base[2];
            bool raised = false;
            float fix[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                top[half] = fmaxf(top[half], __shfl_xor_sync(kFull, top[half], 1));
                top[half] = fmaxf(top[half], __shfl_xor_sync(kFull, top[half], 2));
                const float mn = fmaxf(m[half], top[half] * factor[half]);
                base[half] = mn == -INFINITY ? 0.f : mn - kLift;
                fix[half] = m[half] == -INFINITY ? 1.f : ex2(m[half] - mn);
                raised |= mn > m[half];
                m[half] = mn;
            }
            if (__any_sync(kFull, raised)) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    l[half] *= fix[half];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        o[t][2 * half] *= fix[half];
                        o[t][2 * half + 1] *= fix[half];
                    }
                }
            }
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[t][e] = ex2(fmaf(p[t][e], factor[e >> 1], -base[e >> 1]));
                    l[e >> 1] += p[t][e];
                }
            uint32_t pa[NQ][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = e >> 1, half = e & 1;
                pa[0][e] = pack2<KT>(p[t][2 * half], p[t][2 * half + 1]);
                if constexpr (NQ == 2) pa[1][e] = pack2_rest(p[t][2 * half], p[t][2 * half + 1], pa[0][e]);
            }
            {
                const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c0 = lane >> 4;
#pragma unroll
                for (int t = 0; t < NT; t += 2) {
                    uint32_t b[4];
                    ldsm4t(b, vs + (uint32_t)r * C::kRow + (uint32_t)(((t + c0) ^ (r & 7)) * 16));
                    if constexpr (NQ == 1) {
                        mma16816<KT>(o[t], pa[0], b[0], b[1]);
                        mma16816<KT>(o[t + 1], pa[0], b[2], b[3]);
                    } else {
                        // f32: a product of its own, added here: the tensor cores
                        // cut their additions towards zero, 2^-24 of the sum each
                        // (16000 keys with values about 1 were off by 2.6e-5)
                        float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                        for (int n = NQ - 1; n >= 0; --n) {
                            mma16816<KT>(d[0], pa[n], b[0], b[1]);
                            mma16816<KT>(d[1], pa[n], b[2], b[3]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[t][e] += d[0][e];
                            o[t + 1][e] += d[1][e];
                        }
                    }
                }
            }
        }
        stage = stage + 1 == C::kStages ? 0u : stage + 1;
        const bool last_block = it.blk + 1 == it.blks;
        if (last_block || it.u + 1 >= u1) {
            // the warps' shares of the segment meet in shared memory, 8 rows
            // at a time
            // a segment that starts inside its item leaves a partial; one that
            // starts it joins the shares share + 1 .. last that hold the rest
            const bool leaves = first_blk > 0;
            const int share = my_share(), last = last_block ? share : begin.deal.holder(it.u + (it.blks - 1 - it.blk));
            if (!leaves && !last_block) {
                bool good = true;
                for (int p = share + 1 + tid; p <= last; p += kDcThreads) good &= flag_wait(flags + p, number);
                if (!good) report(a.status, kStatusAttentionWait);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                l[half] += __shfl_xor_sync(kFull, l[half], 1);
                l[half] += __shfl_xor_sync(kFull, l[half], 2);
                if (quad == 0) ml[warp * kDcRows + grp + 8 * half] = make_float2(m[half], l[half]);
            }
            __syncthreads();
            const int rows = min(kDcRows, it.q.n * a.group - it.rt * kDcRows);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (8 * half >= rows) break;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kDcWarps; ++w) top = fmaxf(top, ml[w * kDcRows + grp + 8 * half].x);
                const float mine = m[half] == -INFINITY ? 0.f : ex2(m[half] - top);
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    *(float2 *)(merge + C::at(warp * 8 + grp, 8 * t + 2 * quad)) =
                        make_float2(o[t][2 * half] * mine, o[t][2 * half + 1] * mine);
                __syncthreads();
                constexpr int C4 = D / 4;  // float4 columns of a row
                for (int i = tid; i < min(8, rows - 8 * half) * C4; i += kDcThreads) {
                    const int r8 = i / C4, r = r8 + 8 * half, c = (i % C4) * 4;
                    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                    float big = -INFINITY, den = 0.f;
#pragma unroll
                    for (int w = 0; w < kDcWarps; ++w) big = fmaxf(big, ml[w * kDcRows + r].x);
#pragma unroll
                    for (int w = 0; w < kDcWarps; ++w) {
                        const float4 x = *(const float4 *)(merge + C::at(w * 8 + r8, c));
                        sum.x += x.x; sum.y += x.y; sum.z += x.z; sum.w += x.w;
                        const float2 y = ml[w * kDcRows + r];
                        den += y.x == -INFINITY ? 0.f : y.y * ex2(y.x - big);
                    }
                    if (!leaves) {
                        for (int p = share + 1; p <= last; p += 8) {
                            float pm[8], pl[8];
                            float4 v[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float *part = partials + (size_t)(p + k) * C::kPartial;
                                const bool live = p + k <= last;
                                pm[k] = live ? __ldcg(part + kDcRows * D + r) : -INFINITY;
                                pl[k] = live ? __ldcg(part + kDcRows * D + kDcRows + r) : 0.f;
                                v[k] = live ? __ldcg((const float4 *)(part + r * D + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
                            }
                            float top = big;
#pragma unroll
                            for (int k = 0; k < 8; ++k) top = fmaxf(top, pm[k]);
                            const float fo = big == -INFINITY ? 0.f : ex2(big - top);
                            den *= fo;
                            sum = make_float4(sum.x * fo, sum.y * fo, sum.z * fo, sum.w * fo);
                            big = top;
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float fn = pm[k] == -INFINITY ? 0.f : ex2(pm[k] - top);
                                den += pl[k] * fn;
                                sum = make_float4(sum.x + v[k].x * fn, sum.y + v[k].y * fn, sum.z + v[k].z * fn, sum.w + v[k].w * fn);
                            }
                        }
                        const int row = it.rt * kDcRows + r, token = row / a.group;
                        const bool none = it.q.keys - it.q.n + token + 1 <= 0;
                        const float inv = 1.f / den;
                        const float4 y = none ? make_float4(0.f, 0.f, 0.f, 0.f)
                                              : make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
                        T *out = (T *)a.out + (int64_t)(it.q.row0 + token) * a.out_ld +
                                 (int64_t)(it.h * a.group + row - token * a.group) * D + c;
                        if (store4<T>(out, y)) atomicOr(&bad_rows, 1u << r);
                    } else {
                        float *part = partials + (size_t)share * C::kPartial;
                        *(float4 *)(part + r * D + c) = sum;
                        if (c == 0) {
                            part[kDcRows * D + r] = big;
                            part[kDcRows * D + kDcRows + r] = den;
                        }
                    }
                }
                __syncthreads();
            }
            if (leaves && tid == 0) flag_set(flags + share, number);
            const unsigned bad = bad_rows;
            if (bad) {  // a masked NaN or infinity met the sums: those rows again, without it
                for (int r = warp; r < rows; r += kDcWarps) {
                    if (!(bad >> r & 1u)) continue;
                    const int row = it.rt * kDcRows + r, token = row / a.group;
                    attention_row<T, KT, D>(a, it.q.row0 + token, it.h * a.group + row - token * a.group, it.s, it.q,
                                            merge + warp * D);
                }
                __syncthreads();
                if (tid == 0) bad_rows = 0u;
                __syncthreads();
            }
            fresh = true;
        }
        it.next(plan);
    }
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

// Activations with the 16-bit caches they go with.
template <typename F> cudaError_t by_type(uint32_t type, uint32_t kv_type, int d, const F &f)
{
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
        using T = decltype(t);
        const int pieces = ((a.q_out ? a.heads : 0) + 2 * a.kv_heads) * (d.value / 2 / Elem<T>::kVec), threads = (pieces + 31) / 32 * 32;
        const int block = threads < 64 ? 64 : threads < kAppendThreads ? threads : kAppendThreads;
        // two tokens a CTA from 2048 on: 9600 tokens (bf16, 28/4/128) take 0.95 of
        // what they take with one, (f32, 14/2/64) 0.82; below, one is as fast or faster
        if (a.tokens >= 2048)
            paged_append_kernel<T, decltype(kt), d.value, 2><<<(unsigned)(a.tokens + 1) / 2, block, 0, s>>>(a, turns);
        else
            paged_append_kernel<T, decltype(kt), d.value, 1><<<(unsigned)a.tokens, block, 0, s>>>(a, turns);
        return cudaGetLastError();
    });
}

// A number for a launch's flags that no other launch has and scratch does
// not hold by chance (splitmix64 of a counter; not 0).
static unsigned long long launch_number()
{
    static std::atomic<unsigned long long> count{0x243f6a8885a308d3ull};
    unsigned long long z = count.fetch_add(0x9e3779b97f4a7c15ull);
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    z ^= z >> 31;
    return z ? z : 1;
}

cudaError_t launch_tag(LaunchTag *tag, void *flags, size_t flag_bytes, cudaStream_t s)
{
    *tag = LaunchTag{launch_number(), nullptr};
    if (s == nullptr || s == cudaStreamLegacy) return cudaSuccess;  // never captured
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(s, &status);
    if (e != cudaSuccess || status != cudaStreamCaptureStatusActive) return e;
    static std::atomic<int> used{0};
    const int i = used.load() < kLaunchCounts ? used.fetch_add(1) : kLaunchCounts;
    if (i >= kLaunchCounts) return cudaMemsetAsync(flags, 0, flag_bytes, s);
    void *counts = nullptr;
    e = cudaGetSymbolAddress(&counts, g_launch_count);
    tag->count = (unsigned long long *)counts + i;
    return e;
}

cudaError_t launch_decode_attention(const AttnArgs &a, cudaStream_t s)
{
    return by_type(a.type, a.kv_type, a.head_dim, [&](auto t, auto kt, auto d) {
        using T = decltype(t);
        using KT = decltype(kt);
        constexpr int D = d.value;
        using C = Dc<D>;
        int dev = 0, sms = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(decode_attention_kernel<T, KT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
        // no more CTAs than units there can be, and no partials where an
        // item has one unit at most
        const int64_t blocks = (((int64_t)a.kv.max_pages << a.kv.page_shift) + kDcUnit - 1) / kDcUnit;
        const int64_t tiles = ((int64_t)a.tokens * a.group + kDcRows - 1) / kDcRows + a.sequences;
        const int64_t most = tiles * a.kv_heads * blocks;
        const int ctas = (int)(most < kDcPerSm * sms ? most : kDcPerSm * sms);
        const bool split = ctas > 1 && blocks > 1;
        const size_t bytes = (size_t)ctas * C::kPartial * sizeof(float);
        char *scratch = nullptr;  // a partial and a flag a share
        if (e == cudaSuccess && split) e = stream_alloc((void **)&scratch, bytes + (size_t)ctas * 8, s);
        if (e != cudaSuccess) return e;
        LaunchTag tag{0, nullptr};
        if (split) e = launch_tag(&tag, scratch + bytes, (size_t)ctas * 8, s);
        const DcPlan plan{a.start, a.length, a.sequences, a.tokens, a.kv.max_pages << a.kv.page_shift, a.kv_heads, a.group, divisor(ctas)};
        if (e == cudaSuccess) {
            decode_attention_kernel<T, KT, D><<<(unsigned)ctas, kDcThreads, C::kSmem, s>>>(a, plan, (float *)scratch, (unsigned long long *)(scratch + bytes), tag);
            e = cudaGetLastError();
        }
        const cudaError_t f = stream_free(scratch, s);
        return e != cudaSuccess ? e : f;
    });
}

cudaError_t attention_status_word(unsigned int **word)
{
    static thread_local unsigned int *have[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= 64)) e = cudaErrorInvalidDevice;
    if (e == cudaSuccess && have[dev] == nullptr) e = cudaGetSymbolAddress((void **)&have[dev], g_attention_status);
    if (e == cudaSuccess) *word = have[dev];
    return e;
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
