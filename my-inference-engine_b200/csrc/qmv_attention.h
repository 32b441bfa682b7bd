// Internal interface between the attention entry points
// (qmv_attention_capi.cpp) and their sm_100a kernels (qmv_attention.cu and
// qmv_attention_tc.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace qmv {

enum : uint32_t { kTypeF32 = 0u, kTypeF16 = 1u, kTypeBF16 = 30u };
constexpr int kMaxGroup = 64;  // query heads per key/value head

// Where a sequence's keys and values lie, in elements.  Paged: position p of
// sequence s is row p & (page_size - 1) of page table[s * max_pages +
// (p >> page_shift)].  Packed (table null): row start[s] + p, the position strides
// being k_pos and v_pos.
struct KvView {
    const void *k, *v;
    int64_t k_pos, v_pos;  // between positions
    int64_t page, head;    // between pages, between heads
    const int *table;
    int max_pages, page_shift, page_count;
};

struct AttnArgs {
    uint32_t type, kv_type;
    const void *q;
    void *out;
    int64_t q_ld, out_ld;
    KvView kv;
    const int *start;   // [sequences + 1]
    const int *length;  // [sequences]; null: a sequence's own tokens are its keys
    int sequences, tokens, heads, kv_heads, group, head_dim;
    int max_query;
    float scale;  // multiplies q . k
    unsigned int *status;  // attention_status_word of the device
};

struct AppendArgs {
    uint32_t type, kv_type;
    const void *q, *k, *v;
    void *q_out, *k_out;
    int64_t q_ld, k_ld, v_ld, q_out_ld, k_out_ld;
    KvView kv;  // k / v: the cache's pages (written)
    const int *start, *length;
    int sequences, tokens, heads, kv_heads, head_dim;
    float rope_base;
    unsigned int *status;
};

cudaError_t launch_paged_append(const AppendArgs &a, cudaStream_t s);
// Paged, 16-bit cache: for few rows a sequence over many keys.
cudaError_t launch_decode_attention(const AttnArgs &a, cudaStream_t s);
// Prompts and chunks, on tcgen05.
cudaError_t launch_tc_attention(const AttnArgs &a, cudaStream_t s);

// What a launch's flags carry: a number that no other launch has, and where the
// launch is captured, a count of CTAs on the device that is its own.  (A captured
// launch is one executable graph's, since the scratch it allocates is.)
struct LaunchTag {
    unsigned long long number, *count;
};
// Captured launches beyond the counts clear their flags on the stream instead,
// which costs a replay 2 us.
constexpr int kLaunchCounts = 4096;
cudaError_t launch_tag(LaunchTag *tag, void *flags, size_t flag_bytes, cudaStream_t s);

// Status bits of the attention kernels on the current device.
enum : unsigned int { kStatusBadMetadata = 32u, kStatusAttentionWait = 64u };
cudaError_t attention_status_word(unsigned int **word);
cudaError_t attention_status(unsigned int *out, bool clear);

}  // namespace qmv
