// Causal grouped-query attention on the 5th-generation tensor cores, for
// prompts (packed rows) and for chunks of new tokens over the paged cache.
//
// The query rows of one (sequence, key/value head) are its tokens times its
// group of query heads, so a 128-row MMA tile holds 128 / group tokens with
// all heads that read the same keys: the tile is full for any group, keys are
// fetched once for the group, and the diagonal wastes few keys.  A CTA works
// on two such tiles at once over the same blocks of 128 keys, so that the
// tensor cores multiply for one while the other's softmax runs:
//   S = Q K^T   tcgen05.mma, both operands in shared memory (TMA, 128-byte
//               swizzle), 128 x 128 f32 in tensor memory;
//   softmax     one thread a row: the row of S in registers, running reference
//               m and sum l; P = 2^(S f - m) rounded to the values' 16-bit type
//               (f32: to two or three parts of it) and stored to tensor memory;
//   O += P V    tcgen05.mma, P from tensor memory, V from shared memory.
// S is needed only until it is in registers, so the next scores are multiplied
// while the exponentials run: head_dim 128 has room for one S that the two
// tiles use in turn (S 128 columns, P 2 x 64, O 2 x 128), head_dim 64 for one
// each.  An MMA holds its issuer until the tensor cores take it, so one warp
// issues the QK and another the PV products, and the waits of one hide behind
// the other's work (with one issuer, 1450 of 3500 cycles a block were gaps).
//  (With P over S a
// softmax waited 950 to 1250 of 3250 cycles a block for its next scores; with
// S in halves of 64 keys it did not wait, but the N = 64 MMAs ran at half rate.)
// The reference m is the running maximum, but it is raised only when the
// maximum passes it by kRaise (f32 sums do not care), so O is rescaled a few
// times a row at most.
//
// Where no row of a tile sees the second half of its last block (half of all
// tiles, and every short prompt), 16-bit activations leave it out of the
// softmax and of PV: 61 prompts of 1..64 tokens (f16, 32/8/128) took 34.2 us and
// take 29.6, 13 ragged prompts (bf16, 14/2/64) 126 and 120, and a prompt of 8192
// tokens (bf16, 28/4/128) pays 387 to 393 for the larger code (replayed).  f32 goes
// by halves of a block throughout.
//
// Work is dealt evenly: a tile costs its keys plus a constant, all tiles of
// the launch in order are cut into one equal share per SM at multiples of 128
// keys, and a tile that is cut is joined by the share that holds its beginning.
// So ragged lengths, causal triangles and single long chunks load every SM alike.
#include <cuda.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <atomic>

#include "qmv_attention.cuh"
#include "qmv_internal.h"

namespace qmv {

namespace {

constexpr int kTcKeys = 128;     // keys of a block
constexpr int kTcRows = 128;     // rows of a tile
constexpr int kTcThreads = 384;  // warps 0-3 and 4-7: softmax of a tile each; then
constexpr int kTcQkWarp = 8, kTcPvWarp = 9, kTcLoadVWarp = 11;  // 10: loads Q and K

// T, KT: types of the activations and of the keys and values.
//
// f32 queries and keys meet the tensor cores as pairs of f16, x = hi + lo,
// each row scaled by a power of two that its largest |x| chooses (an element
// is held to 22 bits, or to 2^-39 of that largest one), in the products hi hi,
// lo hi and hi lo.  The weights over f16 pages are pairs of f16 too.  f32
// values meet their weights as three bf16 each (24 bits), in the six products
// above 2^-24: bf16 has f32's exponents, so that values of any size, side by
// side in a row or a column, and weights of any size keep their bits.  (As f16
// pairs scaled by rows, a value of 1e7 cost the other columns 11 of 22 bits.)
template <typename T, typename KT, int D> struct Tc {
    static constexpr int kQ = sizeof(T) == 4 ? 2 : 1;   // parts of Q
    static constexpr int kK = sizeof(KT) == 4 ? 2 : 1;  // parts of K
    static constexpr int kV = sizeof(KT) == 4 ? 3 : 1;  // parts of V
    static constexpr int kP = kV == 3 ? 3 : kQ;         // parts of P
    using MT = typename std::conditional<kQ == 2, __half, T>::type;             // of Q K^T
    using VT = typename std::conditional<kV == 3, __nv_bfloat16, MT>::type;     // of P V
    static constexpr int kSubs = kQ == 2 && D == 128 ? 1 : 2;  // tiles of a CTA: what tensor memory holds
    // What a pair of tiles costs beside its keys, in keys.  Tried on each kind:
    // 16 bits, head_dim 128: a prompt of 8192 tokens takes 400, 399, 393, 393 us
    // with 384, 448, 512, 640, 61 prompts of 1..64 tokens 25.4, 26.3, 26.4,
    // 29.6 us; head_dim 64: 13 ragged prompts 119, 120, 119, 127 us with 256, 288,
    // 320, 384.  f32 over f16 keys: 16 chunks of 1..256 tokens (28/4/128) 108, 97,
    // 92, 92, 93 us with 320, 448, 540, 640, 800, (14/2/64) 45, 45, 45, 47, 47;
    // over f32 keys, head_dim 128: 3 prompts of 400..2000 tokens (28/4) 154, 156,
    // 157, 161, 161 us and one of 3000 390, 382, 384, 387, 395 with 400, 480, 560,
    // 640, 720; head_dim 64 (14/2) 62, 62, 60, 65 and 138, 133, 135, 141 with 224,
    // 288, 336, 400.
    static constexpr int kOver = kK == 2 && D == 64 ? 336 : kK == 2 ? 560 : kQ == 2 ? 540 : D == 64 ? 320 : 512;
    static constexpr uint32_t kTile = 128 * D * 2;  // 128 rows of 16-bit elements
    static constexpr uint32_t kHalf = 128 * 128;    // 128 rows of 64 elements
    static constexpr uint32_t kQTile = kQ * kTile, kKTile = kK * kTile;
    // blocks of K in flight, and pieces of V: a block, or 64 keys of one part
    static constexpr int kSlots = kKTile == 65536 ? 1 : kKTile == 32768 ? 2 : 4;
    static constexpr int kVSlots = kV == 1 ? kSlots : D == 64 ? 10 : 5;
    static constexpr uint32_t kVTile = kV == 1 ? kTile : kTile / 2;
    static constexpr uint32_t kSmem = kSubs * kQTile + kSlots * kKTile + kVSlots * kVTile + 1024;
    // f32 goes by halves of a block: P of 64 keys in parts of 32 columns, and a
    // product of its own for each half, added to the output's sum by the softmax
    // warps.  (The tensor cores cut what an addition leaves behind the 24th bit,
    // and always towards zero: each costs 2^-24 of the sum so far.  With all of a
    // row's keys added there, 16000 keys with values about 1 were off by 2e-4;
    // the plain form in f32 by 1e-7.)  For head_dim 64 the sum is in registers,
    // for 128 in tensor memory behind the product.
    static constexpr uint32_t kPCols = kQ == 2 ? 32u * kP : 64u;
    static constexpr int kSum = kQ == 2 && D == 128 ? D : 0;  // columns of the sum
    // tensor memory columns
    static constexpr int kScores = D == 64 && kK == 1 ? 2 : 1;  // S buffers
    static __host__ __device__ constexpr uint32_t s_col(int x) { return kScores == 2 ? 128u * x : 0u; }
    static __host__ __device__ constexpr uint32_t p_col(int x) { return 128u * kScores + kPCols * x; }
    static __host__ __device__ constexpr uint32_t o_col(int x) { return 128u * kScores + kPCols * kSubs + (uint32_t)(D + kSum) * x; }
    // How far the maximum may pass the reference before it is raised, and how far
    // the weights are lifted, both log2.  bf16 weights have exponents enough.
    // f16 ones are lifted to 2^15.875 (f16 ends at 2^16 - 32): they keep their 11
    // bits down to 2^-27 of the largest, and as pairs 22 bits down to 2^-17 and
    // 2^-39 of the largest below; beside a sink that has most of the weight and
    // little value, those make the output.  (With 8 and 4, a row whose sink had
    // 2^20 times a middling key's weight kept 9 of 22 bits.  A score so large that
    // its rounding passes the end gives an infinity, and that row is computed
    // again.)
    static constexpr float kRaise = !std::is_same<VT, __half>::value ? 8.f : kP == 2 ? 1.f : 2.f;
    static constexpr float kLift = std::is_same<VT, __half>::value ? 15.875f - kRaise : 0.f;
    static_assert(128 * kScores + ((int)kPCols + D + kSum) * kSubs <= 512, "tensor memory");
    static constexpr int kPartial = kSubs * (kTcRows * D + 2 * kTcRows);  // floats: per tile O by column quads, m, l
};

// ------------------------------------------------------------------- PTX

__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(1000u)
        : "memory");
    return ok != 0;
}

// Bounded wait for the phase with the given parity; false when it expired.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity)
{
    if (bar_try(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    for (;;) {
        if (bar_try(bar, parity)) return true;
        if (now_ns() - t0 > kWaitLimitNs) return false;
    }
}

// The same by a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(kFull, bar_wait(bar, parity)); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}

// TMA tile loads (no multicast).
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The MMA warp runs converged, so that descriptors stay in uniform registers;
// one elected lane issues.  (With a single lane in the loop, each MMA took
// 140 cycles to issue, twice what it takes to run.)
__device__ __forceinline__ void commit(uint32_t bar)
{
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

// d (+)= A B over 64 elements of the reduction, both operands in shared
// memory, K-major: 16 elements are 32 bytes, 2 in a descriptor.
__device__ __forceinline__ void mma_ss64(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// The same with A (16-bit pairs, 8 columns for 16 elements) in tensor memory
// and B MN-major: 16 rows of the reduction are 2048 bytes, 128 in a descriptor.
__device__ __forceinline__ void mma_ts64(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile(
        "{\n\t.reg .pred e, p, t;\n\t.reg .b32 a1, a2, a3;\n\t.reg .b64 b1, b2, b3;\n\t"
        "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
        "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}

// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float *v)
{
    uint32_t *r = (uint32_t *)v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}

__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(addr)
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}

// Shared-memory matrix descriptors, 128-byte swizzle (atoms of 8 rows x 128
// bytes, 1024 bytes apart along the rows).  K-major (Q, K): the contiguous
// 64 elements run along the reduction.  MN-major (V): they run along the
// output columns, the second 64 columns `apart` bytes further.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr)
{
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)1u << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t apart)
{
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(apart >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: f32 accumulator, M = 128, N = n, A and B of the
// same 16-bit type, A K-major, B K-major or MN-major.
template <typename KT> __host__ __device__ constexpr uint32_t idesc(int n, bool mn_major)
{
    return (1u << 4) | (std::is_same<KT, __half>::value ? 0u : (1u << 7) | (1u << 10)) | (mn_major ? 1u << 16 : 0u) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Four keys' units; volatile, so that 128 of them are not held in registers.
__device__ __forceinline__ float4 lds4(const float *p)
{
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"((uint32_t)__cvta_generic_to_shared(p)));
    return v;
}

// Two weights as three bf16 each, by cutting: 8 + 8 + 8 bits, exactly (of
// weights above 2^-100).
__device__ __forceinline__ void cut3(float a, float b, uint32_t part[3])
{
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        part[k] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
        if (k == 2) break;
        const float2 rest = __fadd2_rn(make_float2(a, b), make_float2(-__uint_as_float(__float_as_uint(a) & 0xffff0000u),
                                                                     -__uint_as_float(__float_as_uint(b) & 0xffff0000u)));
        a = rest.x;
        b = rest.y;
    }
}

// A warp's 32 f32 rows of Q (rows 32 * quarter .. of the tile) as two f16 rows
// each in swizzled shared memory, the second in the tile behind: x = (hi + lo)
// 2^-e, the largest |x| of a row in [2^14, 2^15) after the shift.  2^-e of each
// lane's own row is returned.  D / 4 lanes take a row, 16 bytes each; rows
// without a token are zeros.  Four loads in flight: more take longer, for the
// size of the code (16, 8, 4: a step of 16 sequences with up to 256 tokens, 14/2/64,
// takes 40.4, 39.4, 39.2 us, 3 prompts of 400..2000 tokens 48.2, 46.7, 46.1).
template <int D> __device__ __forceinline__ float split_rows(const AttnArgs &a, int token_row0, int tokens, int head0, uint32_t tile, int quarter)
{
    constexpr int L = D / 4, R = 32 / L, N = 4;  // lanes a row, rows a load, loads in flight
    const int lane = threadIdx.x & 31, l = lane % L;
    const float per_head = 1.f / (float)a.group;  // (r + 1/2) times it, cut: r / group for r < 128 and groups to 64
    float unit = 1.f;
#pragma unroll 1
    for (int g = 0; g < 32 / R; g += N) {
        float4 v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = 32 * quarter + (g + i) * R + lane / L, token = (int)(((float)r + 0.5f) * per_head);
            v[i] = token < tokens ? *(const float4 *)((const float *)a.q + (int64_t)(token_row0 + token) * a.q_ld +
                                                       (int64_t)(head0 + r - token * a.group) * D + 4 * l)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = 32 * quarter + (g + i) * R + lane / L;
            float big = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
            for (int d = L / 2; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(kFull, big, d));
            const int e = min(max(14 - (int)((__float_as_uint(big) >> 23) & 255u) + 127, kUnitMin), kUnitMax);
            const float up = __uint_as_float((uint32_t)(127 + e) << 23);
            const uint32_t h0 = pack2<__half>(v[i].x * up, v[i].y * up), h1 = pack2<__half>(v[i].z * up, v[i].w * up);
            const uint32_t l0 = pack2_rest(v[i].x * up, v[i].y * up, h0), l1 = pack2_rest(v[i].z * up, v[i].w * up, h1);
            const uint32_t to = tile + (uint32_t)(l / 16) * 16384u + (uint32_t)r * 128u + (uint32_t)((((l / 2) & 7) ^ (r & 7)) * 16 + (l & 1) * 8);
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(h0), "r"(h1) : "memory");
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to + 128u * D * 2u), "r"(l0), "r"(l1) : "memory");
            // to the lane whose row it is: row (g + i) R + k of the warp is lane L k's
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const float u = __shfl_sync(kFull, __uint_as_float((uint32_t)(127 - e) << 23), L * k);
                if (lane == (g + i) * R + k) unit = u;
            }
        }
    }
    return unit;
}

// f32 keys as two f16 planes [part][token][kv_heads * D] and their units (see
// TcMaps): the largest |x| of a row in [2^14, 2^15).  f32 values as three bf16
// planes, each the rounding of what the ones before leave.  A warp a row.
template <int D>
__global__ void __launch_bounds__(256) split_kv_kernel(AttnArgs a, __half *__restrict__ kp, __nv_bfloat16 *__restrict__ vp, float *__restrict__ key_unit)
{
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, rows = a.tokens * a.kv_heads;
    const size_t plane = (size_t)rows * D;
    for (int w = blockIdx.x * 8 + (int)(threadIdx.x >> 5); w < 2 * rows; w += gridDim.x * 8) {
        const bool value = w >= rows;
        const int at = value ? w - rows : w, token = at / a.kv_heads, h = at - token * a.kv_heads;
        const float *x = value ? (const float *)a.kv.v + (int64_t)token * a.kv.v_pos + h * D : (const float *)a.kv.k + (int64_t)token * a.kv.k_pos + h * D;
        float v[E], big = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            v[i] = x[E * lane + i];
            big = fmaxf(big, fabsf(v[i]));
        }
        if (value) {
            __nv_bfloat16 *to = vp + (size_t)at * D + E * lane;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                float2 rest = make_float2(v[i], v[i + 1]);
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    const uint32_t w2 = pack2<__nv_bfloat16>(rest.x, rest.y);
                    *(uint32_t *)(to + k * plane + i) = w2;
                    rest.x -= __uint_as_float(w2 << 16);
                    rest.y -= __uint_as_float(w2 & 0xffff0000u);
                }
            }
            continue;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) big = fmaxf(big, __shfl_xor_sync(kFull, big, d));
        const int top = (int)((__float_as_uint(big) >> 23) & 255u) - 127;
        const int e = min(max(14 - top, kUnitMin), kUnitMax);
        const float up = __uint_as_float((uint32_t)(127 + e) << 23);
        __half *to = kp + (size_t)at * D + E * lane;
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const uint32_t hi = pack2<__half>(v[i] * up, v[i + 1] * up);
            *(uint32_t *)(to + i) = hi;
            *(uint32_t *)(to + plane + i) = pack2_rest(v[i] * up, v[i + 1] * up, hi);
        }
        if (lane == 0) key_unit[(size_t)h * a.tokens + token] = __uint_as_float((uint32_t)(127 - e) << 23);
    }
}

// 32 values of a row, whole 32-byte sectors a store where rows allow.
template <typename T> __device__ __forceinline__ void store32(T *out, const float *o, bool wide)
{
    if (wide) {
#pragma unroll
        for (int i = 0; i < 32; i += 32 / (int)sizeof(T)) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (sizeof(T) == 4)
                    w[j] = __float_as_uint(o[i + j]);
                else
                    w[j] = pack2<T>(o[i + 2 * j], o[i + 2 * j + 1]);
            }
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + i), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += Elem<T>::kVec) Elem<T>::store(out + i, o + i);
    }
}

// ------------------------------------------------------------------ work

struct TcPlan {
    static constexpr int kLeast = 512;  // keys
    const int *start, *length;
    int sequences, tokens, max_keys, kv_heads, over;
    int sub;       // tokens of a tile
    Divisor wide;  // tokens of a CTA's pair of tiles
    Divisor ctas;
    __device__ __forceinline__ Seq seq(int s) const { return load_sequence(start, length, s, tokens, max_keys); }
    // Pair i of a sequence spans over + the keys its last token sees (at
    // least 1) places; the first k pairs of a head span:
    __device__ __forceinline__ long long before(const Seq &q, int k) const
    {
        const long long c = (q.keys > q.n ? q.keys - q.n : 0) + over, all = (long long)k * wide.d;
        return (long long)k * c + (all * (k + 1) >> 1) - (all > q.n ? all - q.n : 0);
    }
    __device__ __forceinline__ int pairs(const Seq &q) const { return (int)__umul64hi((unsigned long long)(q.n + wide.d - 1), wide.magic); }
    __device__ __forceinline__ long long cost(const Seq &q) const { return before(q, pairs(q)) * kv_heads; }
};

// Walks the pairs of tiles in order: sequence, head, pair.  Key block b of a
// pair lies at place origin + over + 128 b; a CTA has the blocks whose places
// fall in its share.
struct TcIter {
    Seq q;
    int s, h, i, pairs, b0, blocks;
    long long origin;
    __device__ __forceinline__ void size(const TcPlan &p)
    {
        const int keys = q.keys - q.n + min((i + 1) * p.wide.d, q.n);
        blocks = keys > 0 ? (keys + kTcKeys - 1) / kTcKeys : 1;
    }
    __device__ __forceinline__ void enter(const TcPlan &p)
    {
        pairs = 0;
        while (s < p.sequences) {
            q = p.seq(s);
            pairs = p.pairs(q);
            if (pairs > 0) break;
            ++s;
        }
    }
    __device__ __forceinline__ void next(const TcPlan &p)
    {
        // (before(i + 1) - before(i), without the products)
        origin += (q.keys > q.n ? q.keys - q.n : 0) + p.over + min((i + 1) * p.wide.d, q.n);
        b0 = 0;
        if (++i == pairs) {
            i = 0;
            if (++h == p.kv_heads) {
                h = 0;
                ++s;
                enter(p);
            }
        }
        if (pairs) size(p);
    }
    // The first block at or behind place u, which is place rel of sequence s_
    // (one with pairs).
    __device__ __forceinline__ void begin(const TcPlan &p, int s_, const Seq &q_, long long rel, long long u)
    {
        s = s_;
        q = q_;
        pairs = p.pairs(q);
        const long long head = p.before(q, pairs);
        h = min(p.kv_heads - 1, (int)((float)rel / (float)head));
        while (h * head > rel) --h;
        while ((h + 1) * head <= rel) ++h;
        rel -= h * head;
        // the last pair i with before(i) <= rel: the root of before's
        // quadratic, then exactly
        const float c = (float)((q.keys > q.n ? q.keys - q.n : 0) + p.over) + 0.5f * (float)p.wide.d;
        i = (int)((sqrtf(c * c + 2.f * (float)p.wide.d * (float)rel) - c) / (float)p.wide.d);
        i = min(max(i, 0), pairs - 1);
        while (i > 0 && p.before(q, i) > rel) --i;
        while (i + 1 < pairs && p.before(q, i + 1) <= rel) ++i;
        origin = u - (rel - p.before(q, i));
        size(p);
        b0 = block_at(p, u);
        if (b0 >= blocks) next(p);
    }
    // The first block at or behind place u.
    __device__ __forceinline__ int block_at(const TcPlan &p, long long u) const
    {
        const long long k = u - origin - p.over;
        return k <= 0 ? 0 : (int)min((k + kTcKeys - 1) / kTcKeys, (long long)blocks);
    }
};

// One tile of a pair: its tokens and key blocks.
struct TcSub {
    int token0, tokens;  // within the sequence's new tokens
    int blocks;          // that any of its rows sees (at least 1 when it has tokens)
    int keys;            // that any of its rows sees
    // no row sees the second half of block b
    __device__ __forceinline__ bool half(int b) const { return keys - b * kTcKeys <= kTcKeys / 2; }
    // halves of blocks that its rows see of blocks 0 .. b1 - 1
    __device__ __forceinline__ int halves(int b1) const
    {
        const int end = min(b1, blocks);
        return 2 * end - (end > 0 && half(end - 1) ? 1 : 0);
    }
    __device__ __forceinline__ TcSub(const TcPlan &p, const TcIter &it, int x)
    {
        token0 = it.i * p.wide.d + x * p.sub;
        tokens = max(0, min(p.sub, it.q.n - token0));
        keys = it.q.keys - it.q.n + token0 + tokens;
        blocks = tokens == 0 ? 0 : keys > 0 ? (keys + kTcKeys - 1) / kTcKeys : 1;
    }
};

struct TcMaps {
    CUtensorMap q, k, v;
    // f32 keys, rows [kv_head][token]: what a key's dot is times (2^-e)
    const float *key_unit;
};


// The output of an uncut pair's row: O from tensor memory times inv (0: a row
// without keys), written where the row has a token (token_row >= 0).  This and
// tc_join are not inlined: their registers would be taken from the softmax
// loop (440 and not 400 us for a prompt of 8192 tokens).
template <typename T, typename KT, int D>
__device__ __noinline__ void tc_store(const AttnArgs &a, uint32_t o_t, float inv, int token_row, int head, int *again)
{
    const bool row = token_row >= 0, wide = (((uintptr_t)a.out | (uintptr_t)(a.out_ld * sizeof(T))) & 31u) == 0;
    T *out = (T *)a.out + (int64_t)(row ? token_row : 0) * a.out_ld + (int64_t)head * D;
    // 0 times a value is 0, or NaN where the value is not finite
    float2 check[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
    for (int c = 0; c < D; c += 64) {
        float o[64];
        tmem_ld32(o_t + c, o);
        tmem_ld32(o_t + c + 32, o + 32);
        wait_ld();
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
            float2 y = __fmul2_rn(make_float2(o[i], o[i + 1]), make_float2(inv, inv));
            if (inv == 0.f) y = make_float2(0.f, 0.f);
            check[i / 2 & 1] = __ffma2_rn(y, make_float2(0.f, 0.f), check[i / 2 & 1]);
            o[i] = y.x;
            o[i + 1] = y.y;
        }
        if (row) {
            store32<T>(out + c, o, wide);
            store32<T>(out + c + 32, o + 32, wide);
        }
    }
    // a masked NaN or infinity may have met the sums
    if (row && !((check[0].x + check[0].y) + (check[1].x + check[1].y) == 0.f)) *again = 1;
}

// The rows of this warp's share that came out not finite, computed again
// without masked keys.  A row may take long (32 keys some microseconds), so
// this comes when no other warp or CTA waits for anything of this warp's any
// more: their limits stay those of a launch without such rows.
template <typename T, typename KT, int D>
__device__ __noinline__ void tc_again(const AttnArgs &a, const TcPlan &plan, TcIter it, long long u1, int x, float *row_q)
{
    const int lane = threadIdx.x & 31, r0 = 32 * ((threadIdx.x >> 5) & 3);
    for (; it.s < plan.sequences && it.block_at(plan, u1) > it.b0; it.next(plan)) {
        if (it.b0 > 0) continue;  // written by an earlier share
        const TcSub me(plan, it, x);
        for (int r = r0; r < min(r0 + 32, me.tokens * a.group); ++r) {
            const int token = r / a.group, head = it.h * a.group + r - token * a.group, row = it.q.row0 + me.token0 + token;
            const T *out = (const T *)a.out + (int64_t)row * a.out_ld + (int64_t)head * D;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < D; e += 32) bad |= !isfinite(Elem<T>::to_float(out[e + lane]));
            if (__any_sync(kFull, bad)) attention_row<T, KT, D>(a, row, head, it.s, it.q, row_q);
        }
    }
}

// What a softmax thread has of its row when its segment ends.
struct TcRow {
    float m, l;
    int keys, token_row, head;
    bool row;  // a row with a token
    bool any;  // the segment holds blocks of this tile
};

// Ends a segment of a cut pair, tile x: the output, or a partial.  Of the shares c0 ..
// last that hold a cut pair, every eighth (c0 + 8 k) joins the seven behind
// it, and c0 joins its seven and the joined eighths: a share waits for later
// ones only, and 37 shares of one long context take 11 + 7 steps and not 36.
constexpr int kJoin = 8;

template <typename T, typename KT, int D>
__device__ __noinline__ void tc_join(const AttnArgs &a, const TcPlan &plan, const TcIter &it, const Deal &deal, int x, uint32_t o_t, TcRow w,
                                     float *partials, unsigned long long *flags, unsigned long long launch, int *again)
{
    using C = Tc<T, KT, D>;
    const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) & 3, r = 32 * quarter + lane, share = my_share();
    const long long first_place = it.origin + plan.over, last_place = first_place + (long long)kTcKeys * (it.blocks - 1);
    const int c0 = it.b0 == 0 ? share : deal.holder(first_place), last = deal.holder(last_place);
    // the shares that this one joins
    const int mine8 = (share - c0) % kJoin == 0 ? min(kJoin - 1, last - share) : 0;
    const int sources = mine8 + (share == c0 ? (last - c0) / kJoin : 0);
    auto source = [&](int k) { return k < mine8 ? share + 1 + k : share + kJoin * (k - mine8 + 1); };
    auto part_of = [&](int p) { return partials + (size_t)p * C::kPartial + (size_t)x * (C::kPartial / C::kSubs); };
    // (every one of them has blocks of the pair: it is kLeast places long, or the
    // last)
    static_assert(TcPlan::kLeast >= kTcKeys, "a share between two block borders would have none");
    unsigned long long *flag = flags + 4 * x + quarter;  // of share 0; a warp's rows are joined by the same warp
    float mine = 1.f;
    if (sources > 0) {
        bool good = true;
        for (int k = lane; k < sources; k += 32) good &= flag_wait(flag + (size_t)source(k) * (4 * C::kSubs), launch);
        if (!good) report(a.status, kStatusAttentionWait);
        __syncwarp();
        float top = w.m, sum = 0.f;
        for (int k0 = 0; k0 < sources; k0 += 4) {
            float pm[4], pl[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float *stat = part_of(source(min(k0 + k, sources - 1))) + kTcRows * D + r;
                pm[k] = k0 + k < sources ? __ldcg(stat) : -INFINITY;
                pl[k] = __ldcg(stat + kTcRows);
            }
            const float before = top;
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, pm[k]);
            sum *= before == -INFINITY ? 0.f : ex2(before - top);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += pm[k] == -INFINITY ? 0.f : pl[k] * ex2(pm[k] - top);
        }
        mine = w.m == -INFINITY ? 0.f : ex2(w.m - top);
        w.m = top;
        w.l = w.l * mine + sum;
    }
    const bool whole = share == c0, none = w.keys <= 0;
    const float scale = whole ? (none ? 0.f : 1.f / w.l) : 1.f;
    const bool wide = (((uintptr_t)a.out | (uintptr_t)(a.out_ld * sizeof(T))) & 31u) == 0;
    T *out = (T *)a.out + (int64_t)w.token_row * a.out_ld + (int64_t)w.head * D;
    float *part = part_of(share);
    float check = 0.f;  // 0 times a value is 0, or NaN where the value is not finite
    if (w.any || sources > 0) {
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float o[32];
            if (w.any) {
                tmem_ld32(o_t + c, o);
                wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
            }
            if (sources > 0) {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= mine;
#pragma unroll 1
                for (int k0 = 0; k0 < sources; k0 += 2) {
                    float f[2];
                    float4 v[2][8];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float *from = part_of(source(min(k0 + k, sources - 1)));
                        const float pm = k0 + k < sources ? __ldcg(from + kTcRows * D + r) : -INFINITY;
                        f[k] = pm == -INFINITY ? 0.f : ex2(pm - w.m);
                        // (where the source has no block of this tile, nothing was written)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            v[k][i] = pm == -INFINITY ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg((const float4 *)(from + ((c / 4 + i) * kTcRows + r) * 4));
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            o[4 * i] = fmaf(v[k][i].x, f[k], o[4 * i]);
                            o[4 * i + 1] = fmaf(v[k][i].y, f[k], o[4 * i + 1]);
                            o[4 * i + 2] = fmaf(v[k][i].z, f[k], o[4 * i + 2]);
                            o[4 * i + 3] = fmaf(v[k][i].w, f[k], o[4 * i + 3]);
                        }
                }
            }
            if (whole) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    o[i] = none ? 0.f : o[i] * scale;
                    check = fmaf(o[i], 0.f, check);
                }
                if (w.row) store32<T>(out + c, o, wide);
            } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *(float4 *)(part + ((c + i) / 4 * kTcRows + r) * 4) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
        }
    }
    if (whole) {
        if (w.row && !(check == 0.f)) *again = 1;  // a masked NaN or infinity may have met the sums
    } else {
        // minus infinity: the row sees no key of the share.  Where it does, a
        // maximum that met only NaN scores, or only minus infinities whose
        // values may be NaN, must not say so.
        part[kTcRows * D + r] = w.keys <= it.b0 * kTcKeys ? -INFINITY : isnan(w.l) ? w.l : fmaxf(w.m, -FLT_MAX);
        part[kTcRows * D + kTcRows + r] = w.l;
        __syncwarp();
        if (lane == 0) flag_set(flag + (size_t)share * (4 * C::kSubs), launch);
    }
}

template <typename T, typename KT, int D>
__global__ void __launch_bounds__(kTcThreads, 1)
tc_attention_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ TcMaps maps, const __grid_constant__ TcPlan plan,
                    float *partials, unsigned long long *flags, LaunchTag tag)
{
    using C = Tc<T, KT, D>;
    using MT = typename C::MT;
    using VT = typename C::VT;
    constexpr int NS = C::kSlots, NV = C::kVSlots, kTcSubs = C::kSubs;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) unsigned long long bars[2 * NS + 2 * NV + 6 * kTcSubs + 3];
    __shared__ uint32_t tmem_slot;
    __shared__ Start<TcIter> begin;
    __shared__ unsigned long long number;
    __shared__ float row_q[4 * kTcSubs][D];
    __shared__ int again[8];  // of each softmax warp: a row of its came out not finite
    // of f32 keys: each key's unit, a copy a warp, this block's and the next one's
    __shared__ __align__(16) float key_of[C::kK == 2 ? 4 * kTcSubs : 1][2][C::kK == 2 ? kTcKeys : 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t smem0 = ((uint32_t)__cvta_generic_to_shared(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = smem0, k_s = smem0 + kTcSubs * C::kQTile, v_s = k_s + NS * C::kKTile;
    const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
    const uint32_t k_full = bar0, k_empty = k_full + 8 * NS, v_full = k_empty + 8 * NS, v_empty = v_full + 8 * NV, q_full = v_empty + 8 * NV, q_empty = q_full + 8 * kTcSubs,
                   s_full = q_empty + 8 * kTcSubs, s_free = s_full + 8 * kTcSubs, p_full = s_free + 8 * kTcSubs,
                   pv_done = p_full + 8 * kTcSubs, tail_bar = pv_done + 8 * kTcSubs, drain_bar = tail_bar + 8;

    if (tid == 32 * kTcLoadVWarp) {
        if (C::kQ == 1) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.q) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.v) : "memory");
    }
    if (tid < 8) again[tid] = 0;
    if (tid == kTcThreads - 1) number = number_of(tag);
    if (tid == 0) {
        for (int i = 0; i < NS; ++i) {
            bar_init(k_full + 8 * i, 1);
            bar_init(k_empty + 8 * i, 1);
        }
        for (int i = 0; i < NV; ++i) {
            bar_init(v_full + 8 * i, 1);
            bar_init(v_empty + 8 * i, 1);
        }
        for (int x = 0; x < kTcSubs; ++x) {
            bar_init(q_full + 8 * x, C::kQ == 2 ? 4 : 1);
            bar_init(q_empty + 8 * x, 1);
            bar_init(s_full + 8 * x, 1);
            bar_init(s_free + 8 * x, 4);
            bar_init(p_full + 8 * x, 4);
            bar_init(pv_done + 8 * x, 1);
        }
        bar_init(tail_bar, 1);
        bar_init(drain_bar, 1);
        bar_init(drain_bar + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kTcQkWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&tmem_slot)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    find_start<kTcThreads>(plan, &begin);
    fence_after();
    const uint32_t tmem = tmem_slot;
    const long long u1 = begin.u1;
    TcIter it = begin.it;
    const int sub = plan.sub;
    // the next segment of this CTA: blocks [it.b0, b1) of the pair
    auto segment = [&](int *b1) {
        if (it.s >= plan.sequences) return false;
        *b1 = it.block_at(plan, u1);
        return *b1 > it.b0;
    };
    bool ok = true;
    int b1 = 0;

    if (warp < 8) {
        // --------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int x = warp >> 2, quarter = warp & 3, r = 32 * quarter + lane;
        const uint32_t lanes = tmem + ((uint32_t)(32 * quarter) << 16);
        const uint32_t s_t = lanes + C::s_col(x), p_t = lanes + C::p_col(x), o_t = lanes + C::o_col(x);
        uint32_t done = 0, seen = 0;  // of this tile slot: blocks (f32: halves) handed over so far, and f32 blocks
        // f32 keys: units of this lane's keys (4 lane ..) of block b
        auto units_of = [&](int b, float u[4]) {
            const int64_t at = (int64_t)it.h * a.tokens + it.q.row0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = b * kTcKeys + 4 * lane + i;
                u[i] = j < it.q.keys ? __ldg(maps.key_unit + at + j) : 1.f;
            }
        };
        for (; x < kTcSubs && ok && segment(&b1); it.next(plan)) {
            const TcSub me(plan, it, x);
            const int end = min(b1, me.blocks), token = r / a.group;
            const bool row = token < me.tokens;
            const int keys = it.q.keys - it.q.n + me.token0 + token + 1;
            // rows without a token run along unmasked and are never written
            const int lim = row ? max(keys, 0) : 0x7fffffff;
            const int head = it.h * a.group + r - token * a.group, token_row = it.q.row0 + me.token0 + token;
            float f = row ? a.scale * kLog2e : 0.f;
            if constexpr (C::kQ == 2) {
                // this thread's row of Q as two f16 rows; the QK products of
                // the tile before have ended, since their scores were read
                if (end > it.b0) {
                    f *= split_rows<D>(a, it.q.row0 + me.token0, me.tokens, it.h * a.group, q_s + x * C::kQTile, quarter);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) bar_arrive(q_full + 8 * x);
                }
            }
            float m = -INFINITY, l = 0.f;
            float next_units[4];
            if constexpr (C::kK == 2)
                if (end > it.b0) units_of(it.b0, next_units);
            // 16 bits: block b, of its keys the first N
            auto block = [&](const int b, auto cols) {
                constexpr int N = decltype(cols)::value;
                if (!warp_wait(s_full + 8 * x, done & 1)) return false;
                fence_after();
                float s[N];
#pragma unroll
                for (int i = 0; i < N / 32; ++i) tmem_ld32(s_t + 32 * i, s + 32 * i);
                wait_ld();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(s_free + 8 * (C::kScores == 2 ? x : 0));
                const int j0 = b * kTcKeys;
                if (__any_sync(kFull, j0 + N > lim)) {
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (j0 + i >= lim) s[i] = -INFINITY;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < N; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f;
                const bool raise = __any_sync(kFull, mx > m + (m == -INFINITY ? 0.f : C::kRaise));
                // P and O as the block before this one left them
                if (done > 0) {
                    if (!warp_wait(pv_done + 8 * x, (done - 1) & 1)) return false;
                    fence_after();
                }
                if (raise) {
                    const float mn = fmaxf(m, mx), fix = m == -INFINITY ? 0.f : ex2(m - mn);
                    m = mn;
                    l *= fix;
                    if (b > it.b0) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            tmem_ld32(o_t + c, o);
                            wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= fix;
                            tmem_st32(o_t + c, (const uint32_t *)o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.f : m - C::kLift;
                const float2 f2 = make_float2(f, f), n2 = make_float2(-base, -base);
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < N / 64; ++h) {
                    uint32_t p[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int j = 2 * (32 * h + i);
                        const float2 e = __ffma2_rn(make_float2(s[j], s[j + 1]), f2, n2), w = make_float2(ex2(e.x), ex2(e.y));
                        sum[i & 1] = __fadd2_rn(sum[i & 1], w);
                        p[i] = pack2<VT>(w.x, w.y);
                    }
                    tmem_st32(p_t + 32 * h, p);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(p_full + 8 * x);
                ++done;
                return true;
            };
            // f32: block b, by halves; the output's sum before them
            constexpr bool kInRegisters = C::kQ == 2 && C::kSum == 0;
            float o_sum[kInRegisters ? 64 : 1];
            constexpr auto kAt = [](int column) { return kInRegisters ? column : 0; };
            bool summed = false;  // there is one
            uint32_t left = 0;    // products not in it yet
            auto add_product = [&](float fix, bool raise) {
                if (left == 0) return true;
                if (!warp_wait(pv_done + 8 * x, (done - 1) & 1)) return false;
                fence_after();
                left = 0;
                if constexpr (C::kSum == 0) {
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        float o[32];
                        tmem_ld32(o_t + c, o);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o_sum[kAt(c + i)] += o[i];  // (in pairs 2 us slower)
                    }
                    if (raise) {
#pragma unroll
                        for (int i = 0; i < 64; ++i) o_sum[kAt(i)] *= fix;
                    }
                } else {
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32], to[32];
                        tmem_ld32(o_t + c, o);
                        tmem_ld32(o_t + D + c, to);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 y = make_float2(o[i], o[i + 1]), z = summed ? __fadd2_rn(make_float2(to[i], to[i + 1]), y) : y;
                            to[i] = z.x;
                            to[i + 1] = z.y;
                        }
                        if (raise) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) to[i] *= fix;
                        }
                        tmem_st32(o_t + D + c, (const uint32_t *)to);
                    }
                    summed = true;
                }
                return true;
            };
            auto block_by_halves = [&](const int b) {
                if (!warp_wait(s_full + 8 * x, seen++ & 1)) return false;
                fence_after();
                float *unit = key_of[C::kK == 2 ? warp : 0][C::kK == 2 ? b & 1 : 0];
                if constexpr (C::kK == 2) {
                    *(float4 *)(unit + 4 * lane) = make_float4(next_units[0], next_units[1], next_units[2], next_units[3]);
                    __syncwarp();
                    if (b + 1 < end) units_of(b + 1, next_units);
                }
#pragma unroll 1
                for (int g = 0; g < 2; ++g) {
                    const bool last = g == 1 || me.half(b);
                    float s[64];
                    tmem_ld32(s_t + 64 * g, s);
                    tmem_ld32(s_t + 64 * g + 32, s + 32);
                    wait_ld();
                    if (last) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(s_free + 8 * (C::kScores == 2 ? x : 0));
                    }
                    const int j0 = b * kTcKeys + 64 * g;
                    if constexpr (C::kK == 2) {
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            const float4 u = lds4(unit + 64 * g + i);
                            const float2 lo = __fmul2_rn(make_float2(s[i], s[i + 1]), make_float2(u.x, u.y)), hi = __fmul2_rn(make_float2(s[i + 2], s[i + 3]), make_float2(u.z, u.w));
                            s[i] = lo.x;
                            s[i + 1] = lo.y;
                            s[i + 2] = hi.x;
                            s[i + 3] = hi.y;
                        }
                    }
                    if (__any_sync(kFull, j0 + 64 > lim)) {
#pragma unroll
                        for (int i = 0; i < 64; ++i)
                            if (j0 + i >= lim) s[i] = -INFINITY;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 64; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
                    const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f;
                    const bool raise = __any_sync(kFull, mx > m + (m == -INFINITY ? 0.f : C::kRaise));
                    float fix = 1.f;
                    if (raise) {
                        const float mn = fmaxf(m, mx);
                        fix = m == -INFINITY ? 0.f : ex2(m - mn);
                        m = mn;
                        l *= fix;
                    }
                    if (C::kP == 3 && !add_product(fix, raise)) return false;
                    const float base = m == -INFINITY ? 0.f : m - C::kLift;
                    const float2 f2 = make_float2(f, f), n2 = make_float2(-base, -base);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t p[C::kP][16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int j = 2 * (16 * h + i);
                            const float2 e = __ffma2_rn(make_float2(s[j], s[j + 1]), f2, n2), w = make_float2(ex2(e.x), ex2(e.y));
                            sum[i & 1] = __fadd2_rn(sum[i & 1], w);
                            if constexpr (C::kP == 3) {
                                uint32_t part[3];
                                cut3(w.x, w.y, part);
#pragma unroll
                                for (int k = 0; k < 3; ++k) p[C::kP == 3 ? k : 0][i] = part[k];
                            } else {
                                p[0][i] = pack2<VT>(w.x, w.y);
                                p[C::kP - 1][i] = pack2_rest(w.x, w.y, p[0][i]);
                            }
                        }
                        if (C::kP == 2 && h == 0 && !add_product(fix, raise)) return false;
#pragma unroll
                        for (int k = 0; k < C::kP; ++k) tmem_st16(p_t + 32 * k + 16 * h, p[k]);
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(p_full + 8 * x);
                    ++done;
                    left = 1;
                    if (last) break;
                }
                return true;
            };
            if constexpr (C::kQ == 2) {
#pragma unroll
                for (float &y : o_sum) y = 0.f;
#pragma unroll 1
                for (int b = it.b0; ok && b < end; ++b) ok = block_by_halves(b);
            } else {
                // the last block may go by halves; in a loop of its own, since a branch
                // within the loop cost a long prompt another 1 to 4 per cent
                const bool half = end > it.b0 && me.half(end - 1);
                const int full = end - (half ? 1 : 0);
#pragma unroll 1
                for (int b = it.b0; ok && b < full; ++b) ok = block(b, std::integral_constant<int, 128>{});
                if (ok && half) ok = block(end - 1, std::integral_constant<int, 64>{});
            }
            if (!ok) break;
            if (me.tokens == 0) continue;
            const bool any = end > it.b0;  // this segment holds blocks of this tile
            if (any) {
                if constexpr (C::kQ == 2) {
                    if (!(ok = add_product(1.f, false))) break;
                    if constexpr (C::kSum == 0) {
#pragma unroll
                        for (int c = 0; c < 64; c += 32) tmem_st32(o_t + c, (const uint32_t *)(o_sum + kAt(c)));
                    }
                    wait_st();
                } else {
                    if (!(ok = warp_wait(pv_done + 8 * x, (done - 1) & 1))) break;
                    fence_after();
                }
            }
            if (it.b0 > 0 || b1 < it.blocks) {
                tc_join<T, KT, D>(a, plan, it, begin.deal, x, o_t + C::kSum, TcRow{m, l, keys, token_row, head, row, any}, partials, flags, number, again + warp);
            } else {
                tc_store<T, KT, D>(a, o_t + C::kSum, keys <= 0 ? 0.f : 1.f / l, row ? token_row : -1, head, again + warp);
            }
            fence_before();
        }
        __syncwarp();
        if (ok && *(volatile int *)(again + warp)) tc_again<T, KT, D>(a, plan, begin.it, u1, x, row_q[warp]);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        uint32_t slot = 0, phase = 0;  // of this warp's next block of K or V
        const uint32_t slots = warp == kTcPvWarp || warp == kTcLoadVWarp ? NV : NS;
        auto step = [&]() {
            if (++slot == slots) {
                slot = 0;
                phase ^= 1;
            }
        };
        if (warp == kTcQkWarp) {
            // ----------------------------------------------------- S = Q K^T
            constexpr uint32_t kId = idesc<MT>(128, false);
            const uint32_t tm = __shfl_sync(kFull, tmem, 0);
            uint32_t q_phase[2] = {0, 0}, s_phase[2] = {1, 1};  // s_phase: of each S buffer
            for (; ok && segment(&b1); it.next(plan)) {
                int end[2];  // of the blocks of each tile
#pragma unroll
                for (int x = 0; x < kTcSubs; ++x) end[x] = min(b1, TcSub(plan, it, x).blocks);
                for (int b = it.b0; b < b1; ++b) {
                    if (!(ok = warp_wait(k_full + 8 * slot, phase))) break;
                    const uint64_t kb = desc_k(k_s + __shfl_sync(kFull, slot, 0) * C::kKTile);
#pragma unroll
                    for (int x = 0; x < kTcSubs; ++x) {
                        if (!ok || b >= end[x]) continue;
                        if (b == it.b0) {
                            ok = warp_wait(q_full + 8 * x, q_phase[x]);
                            q_phase[x] ^= 1;
                        }
                        constexpr int kBuf = C::kScores - 1;
                        if (!ok || !(ok = warp_wait(s_free + 8 * (kBuf * x), s_phase[kBuf * x]))) continue;
                        s_phase[kBuf * x] ^= 1;
                        fence_after();
                        const uint64_t qa = desc_k(q_s + x * C::kQTile);
                        constexpr uint32_t part = C::kTile >> 4;
                        // small products first: each addition rounds to the
                        // sum so far
                        if constexpr (C::kQ == 2) {
#pragma unroll
                            for (int k = 0; k < D / 64; ++k) {
                                const uint32_t at = k * (C::kHalf >> 4);
                                mma_ss64(tm + C::s_col(x), qa + part + at, kb + at, kId, k != 0);
                                if constexpr (C::kK == 2) mma_ss64(tm + C::s_col(x), qa + at, kb + part + at, kId, 1u);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < D / 64; ++k) {
                            const uint32_t at = k * (C::kHalf >> 4);
                            mma_ss64(tm + C::s_col(x), qa + at, kb + at, kId, C::kQ == 2 || k != 0);
                        }
                        commit(s_full + 8 * x);
                        if (b + 1 == end[x]) commit(q_empty + 8 * x);
                    }
                    if (!ok) break;
                    commit(k_empty + 8 * slot);
                    step();
                }
            }
            if (!ok) {  // let what was issued end before tensor memory is given back
                commit(drain_bar);
                bar_wait(drain_bar, 0);
            }
        } else if (warp == kTcPvWarp) {
            // ------------------------------------------------------ O += P V
            constexpr uint32_t kId = idesc<VT>(D, true);
            const uint32_t tm = __shfl_sync(kFull, tmem, 0);
            uint32_t p_phase[2] = {0, 0};
            for (; ok && segment(&b1); it.next(plan)) {
                int end[2];
                bool half[2];
#pragma unroll
                for (int x = 0; x < kTcSubs; ++x) {
                    const TcSub me(plan, it, x);
                    end[x] = min(b1, me.blocks);
                    half[x] = me.half(end[x] - 1);
                }
                constexpr uint32_t rows64 = 64 * 128 >> 4;
                if constexpr (C::kQ == 2) {
                    // f32: a product for each 64 keys
                    int upto[2] = {0, 0};
#pragma unroll
                    for (int x = 0; x < kTcSubs; ++x) upto[x] = TcSub(plan, it, x).halves(b1);
                    for (int g = 2 * it.b0; ok && g < (C::kV == 3 ? max(upto[0], upto[1]) : 2 * b1); ++g) {
                        uint64_t vb[3];
                        const int left = it.q.keys - 64 * g;
                        uint32_t at[3];
                        if constexpr (C::kV == 1) {
                            if ((g & 1) == 0 && !(ok = warp_wait(v_full + 8 * slot, phase))) break;
                            vb[0] = desc_mn(v_s + __shfl_sync(kFull, slot, 0) * C::kVTile, C::kHalf) + (g & 1) * rows64;
                        }
                        // the values' three parts, a slot each
#pragma unroll
                        for (int c = 0; c < (C::kV == 3 ? 3 : 0); ++c) {
                            if (!ok || !(ok = warp_wait(v_full + 8 * slot, phase))) continue;
                            at[c] = slot;
                            const uint32_t to = v_s + __shfl_sync(kFull, slot, 0) * C::kVTile;
                            vb[c] = desc_mn(to, 64 * 128);
                            // the rows behind the last value: zeros, so that no NaN of
                            // another sequence meets a weight of 0
                            if (left < 64) {
                                for (int row = max(0, left) + (lane >> 3); row < 64; row += 4)
#pragma unroll
                                    for (int i = 0; i < D / 64; ++i)
                                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to + i * 8192u + (uint32_t)row * 128u + (lane & 7) * 16u), "r"(0u) : "memory");
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                                __syncwarp();
                            }
                            step();
                        }
#pragma unroll
                        for (int x = 0; x < kTcSubs; ++x) {
                            if (!ok || g >= upto[x]) continue;
                            if (!(ok = warp_wait(p_full + 8 * x, p_phase[x]))) continue;
                            p_phase[x] ^= 1;
                            fence_after();
                            const uint32_t pt = tm + C::p_col(x), ot = tm + C::o_col(x);
                            if constexpr (C::kV == 3) {
                                // the products of the values' parts and the weights' above 2^-24, small ones first
                                mma_ts64(ot, pt + 64u, vb[0], kId, 0u);
                                mma_ts64(ot, pt + 32u, vb[1], kId, 1u);
                                mma_ts64(ot, pt, vb[2], kId, 1u);
                                mma_ts64(ot, pt + 32u, vb[0], kId, 1u);
                                mma_ts64(ot, pt, vb[1], kId, 1u);
                            } else {
                                mma_ts64(ot, pt + 32u, vb[0], kId, 0u);
                            }
                            mma_ts64(ot, pt, vb[0], kId, 1u);
                            commit(pv_done + 8 * x);
                        }
                        if (!ok) break;
                        if constexpr (C::kV == 3) {
#pragma unroll
                            for (int c = 0; c < 3; ++c) commit(v_empty + 8 * at[c]);
                        } else if (g & 1) {
                            commit(v_empty + 8 * slot);
                            step();
                        }
                    }
                }
                for (int b = it.b0; C::kQ == 1 && b < b1; ++b) {
                    if (!(ok = warp_wait(v_full + 8 * slot, phase))) break;
                    const uint64_t vb = desc_mn(v_s + __shfl_sync(kFull, slot, 0) * C::kVTile, C::kHalf);
#pragma unroll
                    for (int x = 0; x < kTcSubs; ++x) {
                        if (!ok || b >= end[x]) continue;
                        if (!(ok = warp_wait(p_full + 8 * x, p_phase[x]))) continue;
                        p_phase[x] ^= 1;
                        fence_after();
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (h == 1 && b + 1 == end[x] && half[x]) break;
                            mma_ts64(tm + C::o_col(x), tm + C::p_col(x) + 32u * h, vb + h * rows64, kId, h != 0 || b != it.b0);
                        }
                        commit(pv_done + 8 * x);
                    }
                    if (!ok) break;
                    commit(v_empty + 8 * slot);
                    step();
                }
            }
            if (!ok) {
                commit(drain_bar + 8);
                bar_wait(drain_bar + 8, 0);
            }
        } else {
            // ------------------------------------------------------- loads
            const bool values = warp == kTcLoadVWarp;
            const uint32_t full = values ? v_full : k_full, empty = values ? v_empty : k_empty, tiles = values ? v_s : k_s;
            const CUtensorMap *map = values ? &maps.v : &maps.k;
            const bool paged = a.kv.table != nullptr;
            const int page_size = paged ? 1 << a.kv.page_shift : kTcKeys, piece = min(page_size, kTcKeys), pieces = kTcKeys / piece;
            const uint32_t q_bytes = (uint32_t)(sub * a.group) * D * 2;
            uint32_t issued = 0, q_phase[2] = {1, 1}, tail_phase = 0;
            phase = 1;  // of the empty barriers
            // page of the piece that this lane copies of block b
            auto page_of = [&](int b) {
                const int j = b * kTcKeys + lane * piece;
                if (!paged || lane >= pieces || j >= it.q.keys) return -1;
                const int page = __ldg(a.kv.table + (int64_t)it.s * a.kv.max_pages + (j >> a.kv.page_shift));
                if (page >= 0 && page < a.kv.page_count) return page;
                report(a.status, kStatusBadMetadata);
                return a.kv.page_count;  // outside the map: zeros
            };
            for (; ok && segment(&b1); it.next(plan)) {
                if (!values && C::kQ == 1) {
                    for (int x = 0; ok && x < kTcSubs; ++x) {
                        const TcSub me(plan, it, x);
                        if (min(b1, me.blocks) <= it.b0) continue;
                        if (!(ok = warp_wait(q_empty + 8 * x, q_phase[x]))) break;
                        q_phase[x] ^= 1;
                        if (lane == 0) {
                            bar_expect(q_full + 8 * x, q_bytes);
#pragma unroll
                            for (int c = 0; c < D / 64; ++c)
                                tma3(q_s + x * C::kQTile + c * C::kHalf, &maps.q, 64 * c, it.h * a.group, it.q.row0 + me.token0, q_full + 8 * x);
                        }
                    }
                }
                if constexpr (C::kV == 3) {
                    if (values) {  // 64 keys of one part after another
                        int upto = 0;
                        for (int x = 0; x < kTcSubs; ++x) upto = max(upto, TcSub(plan, it, x).halves(b1));
                        for (int u = 6 * it.b0; ok && u < 3 * upto; ++u) {
                            if (!(ok = warp_wait(empty + 8 * slot, phase))) break;
                            if (lane == 0) {
                                bar_expect(full + 8 * slot, C::kVTile);
#pragma unroll
                                for (int c = 0; c < D / 64; ++c)
                                    tma4(tiles + slot * C::kVTile + c * 8192u, map, 64 * c, it.h, it.q.row0 + 64 * (u / 3), u % 3, full + 8 * slot);
                            }
                            ++issued;
                            step();
                        }
                        continue;
                    }
                }
                int page = page_of(it.b0);
                for (int b = it.b0; ok && b < b1; ++b) {
                    const int page_next = b + 1 < b1 ? page_of(b + 1) : -1;
                    if (!(ok = warp_wait(empty + 8 * slot, phase))) break;
                    const int j0 = b * kTcKeys, left = it.q.keys - j0;
                    // the rows behind the last value: zeros, so that no stale
                    // NaN meets a weight of 0
                    const bool tail = values && left < kTcKeys;
                    const uint32_t bar = tail ? tail_bar : full + 8 * slot, dst = tiles + slot * C::kKTile;
                    const int live = paged ? min(pieces, max(0, (left + piece - 1) / piece)) : 1;
                    if (lane == 0) {
                        if (live > 0)
                            bar_expect(bar, (uint32_t)(live * piece) * D * 2 * C::kK);
                        else if (!tail)
                            bar_arrive(bar);
                    }
                    __syncwarp();
                    if (lane < live) {
#pragma unroll
                        for (int c = 0; c < D / 64 * C::kK; ++c) {
                            const uint32_t to = dst + c * C::kHalf + (uint32_t)(lane * piece) * 128u;
                            const int x0 = 64 * (c % (D / 64)), part = c / (D / 64);
                            if (paged)
                                tma4(to, map, x0, it.h, (j0 + lane * piece) & (page_size - 1), page, bar);
                            else
                                tma4(to, map, x0, it.h, it.q.row0 + j0, part, bar);
                        }
                    }
                    if (tail) {
                        if (live > 0) {
                            if (!(ok = warp_wait(tail_bar, tail_phase))) break;
                            tail_phase ^= 1;
                        }
                        for (int row = max(0, left) + (lane >> 3); row < kTcKeys; row += 4)
#pragma unroll
                            for (int c = 0; c < D / 64 * C::kK; ++c)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + c * C::kHalf + (uint32_t)row * 128u + (lane & 7) * 16u),
                                             "r"(0u)
                                             : "memory");
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) bar_arrive(full + 8 * slot);
                    }
                    page = page_next;
                    ++issued;
                    step();
                }
            }
            if (!ok) {  // copies in flight land before the CTA ends
                const uint32_t from = issued > slots ? issued - slots : 0;
                for (uint32_t i = from; i < issued; ++i) bar_wait(full + 8 * (i % slots), (i / slots) & 1);
                for (int x = 0; !values && C::kQ == 1 && x < kTcSubs; ++x) bar_wait(q_full + 8 * x, q_phase[x]);
            }
        }
    }
    if (blockIdx.x == 0) check_metadata(a.status, a.start, a.length, a.sequences, a.tokens, plan.max_keys);
    if (!ok && lane == 0) report(a.status, kStatusAttentionWait);
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == kTcQkWarp) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// ---------------------------------------------------------------- launch

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encode_tiled(EncodeTiled *fn)
{
    static std::atomic<EncodeTiled> have{nullptr};  // the same for every thread that looks it up
    if (have.load(std::memory_order_relaxed) == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
        if (e != cudaSuccess) return e;
        if (found != cudaDriverEntryPointSuccess || p == nullptr) return cudaErrorNotSupported;
        have.store((EncodeTiled)p, std::memory_order_relaxed);
    }
    *fn = have.load(std::memory_order_relaxed);
    return cudaSuccess;
}

// 64-element wide boxes of 16-bit elements, 128-byte swizzle, zeros outside.
template <typename KT>
cudaError_t make_map(CUtensorMap *map, const void *base, int rank, const cuuint64_t *dims, const int64_t *strides, const cuuint32_t *box)
{
    EncodeTiled encode = nullptr;
    const cudaError_t e = encode_tiled(&encode);
    if (e != cudaSuccess) return e;
    cuuint64_t bytes[3];
    const cuuint32_t ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank - 1; ++i) bytes[i] = (cuuint64_t)strides[i] * 2;
    const CUresult r = encode(map, std::is_same<KT, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                              (cuuint32_t)rank, const_cast<void *>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, typename KT, int D> cudaError_t launch(const AttnArgs &a, cudaStream_t s)
{
    using C = Tc<T, KT, D>;
    using MT = typename C::MT;
    using VT = typename C::VT;
    const int sub = kTcRows / a.group;
    const bool paged = a.kv.table != nullptr;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tc_attention_kernel<T, KT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t keys = paged ? (int64_t)a.kv.max_pages << a.kv.page_shift : a.tokens, blocks = (keys + kTcKeys - 1) / kTcKeys;
    const int64_t pairs = a.tokens / (sub * C::kSubs) + a.sequences, most = pairs * a.kv_heads * blocks;
    const int ctas = (int)(most < sms ? most : sms);
    const bool split = ctas > 1 && blocks > 1;
    // scratch: a partial a share | flags | planes of K | of V | units of K
    const size_t part_bytes = split ? (size_t)ctas * C::kPartial * sizeof(float) : 0, flag_bytes = split ? (size_t)ctas * 4 * C::kSubs * 8 : 0;
    const size_t plane_at = (part_bytes + flag_bytes + 127) & ~(size_t)127, rows = (size_t)a.tokens * a.kv_heads;
    const size_t key_bytes = rows * D * 2 * C::kK, value_bytes = rows * D * 2 * C::kV;
    char *scratch = nullptr;
    if (split || C::kK == 2) e = stream_alloc((void **)&scratch, plane_at + (C::kK == 2 ? key_bytes + value_bytes + rows * 4 : 0), s);
    if (e != cudaSuccess) return e;
    float *partials = split ? (float *)scratch : nullptr;
    unsigned long long *flags = (unsigned long long *)(scratch + part_bytes);
    LaunchTag tag{0, nullptr};
    if (split) e = launch_tag(&tag, flags, flag_bytes, s);
    TcMaps maps{};
    const void *k = a.kv.k, *v = a.kv.v;
    if constexpr (C::kK == 2) {
        __half *kp = (__half *)(scratch + plane_at);
        __nv_bfloat16 *vp = (__nv_bfloat16 *)(scratch + plane_at + key_bytes);
        float *units = (float *)(scratch + plane_at + key_bytes + value_bytes);
        const size_t want = (2 * rows + 7) / 8, cap = (size_t)sms * 8;
        if (e == cudaSuccess) {
            split_kv_kernel<D><<<(unsigned)(want < cap ? want : cap), 256, 0, s>>>(a, kp, vp, units);
            e = cudaGetLastError();
        }
        k = kp;
        v = vp;
        maps.key_unit = units;
    }
    if constexpr (C::kQ == 1) {
        const cuuint64_t qd[3] = {(cuuint64_t)D, (cuuint64_t)a.heads, (cuuint64_t)a.tokens};
        const int64_t qs[2] = {D, a.q_ld};
        const cuuint32_t qb[3] = {64, (cuuint32_t)a.group, (cuuint32_t)sub};
        if (e == cudaSuccess) e = make_map<MT>(&maps.q, a.q, 3, qd, qs, qb);
    }
    const int page_size = paged ? 1 << a.kv.page_shift : kTcKeys;
    cuuint64_t kd[4] = {(cuuint64_t)D, (cuuint64_t)a.kv_heads, paged ? (cuuint64_t)page_size : (cuuint64_t)a.tokens,
                        paged ? (cuuint64_t)a.kv.page_count : (cuuint64_t)C::kK};
    int64_t ks[3] = {a.kv.head, a.kv.k_pos, paged ? a.kv.page : a.kv.k_pos}, vs[3] = {a.kv.head, a.kv.v_pos, paged ? a.kv.page : a.kv.v_pos};
    if constexpr (C::kK == 2) {
        ks[0] = vs[0] = D;
        ks[1] = vs[1] = (int64_t)a.kv_heads * D;
        ks[2] = vs[2] = (int64_t)rows * D;
    }
    cuuint32_t kb[4] = {64, 1, (cuuint32_t)(page_size < kTcKeys ? page_size : kTcKeys), 1};
    if (e == cudaSuccess) e = make_map<MT>(&maps.k, k, 4, kd, ks, kb);
    if constexpr (C::kV == 3) {
        kd[3] = 3;
        kb[2] = 64;
    }
    if (e == cudaSuccess) e = make_map<VT>(&maps.v, v, 4, kd, vs, kb);
    const TcPlan plan{a.start, a.length, a.sequences, a.tokens, paged ? a.kv.max_pages << a.kv.page_shift : 0x7fffffff, a.kv_heads, C::kOver,
                      sub, divisor(sub * C::kSubs), divisor(ctas)};
    if (e == cudaSuccess) {
        tc_attention_kernel<T, KT, D><<<(unsigned)ctas, kTcThreads, C::kSmem, s>>>(a, maps, plan, partials, flags, tag);
        e = cudaGetLastError();
    }
    const cudaError_t f = stream_free(scratch, s);
    return e != cudaSuccess ? e : f;
}

}  // namespace

cudaError_t launch_tc_attention(const AttnArgs &a, cudaStream_t s)
{
    const bool wide = a.head_dim == 128;
    if (a.type == kTypeF32 && a.kv_type == kTypeF32) return wide ? launch<float, float, 128>(a, s) : launch<float, float, 64>(a, s);
    if (a.type == kTypeF32 && a.kv_type == kTypeF16) return wide ? launch<float, __half, 128>(a, s) : launch<float, __half, 64>(a, s);
    if (a.type == kTypeF16 && a.kv_type == kTypeF16) return wide ? launch<__half, __half, 128>(a, s) : launch<__half, __half, 64>(a, s);
    if (a.type == kTypeBF16 && a.kv_type == kTypeBF16)
        return wide ? launch<__nv_bfloat16, __nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, __nv_bfloat16, 64>(a, s);
    return cudaErrorInvalidValue;
}

}  // namespace qmv
