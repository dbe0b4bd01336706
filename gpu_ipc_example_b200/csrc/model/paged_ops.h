// Host entry points of paged serving: requests of different lengths in one batch, their keys and values in pages of one cache
// [pages, hkv, page, 128] that a block table [requests, width] strings together.  All stream-ordered, no allocation inside, nothing
// read back: lengths live on the GPU, so that a step can be captured.  No counterpart in the reference (it has no model code).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime_api.h>

#include "../common/types.h"

namespace b200ipc {

constexpr int kPagedMaxRequests = 8192;  // of one block table

// What paged_extend and paged_trim found (bits).  With any of them set, nothing has changed.
constexpr int kPagedNoPages = 1;   // extend: the free list has fewer pages than are needed; trim: it has no room for what comes back
constexpr int kPagedTooLong = 2;   // extend: a request outgrows its row of the table; trim: a length to keep is above the present one
constexpr int kPagedTooMany = 4;   // extend: more new tokens than rows
constexpr int kPagedNegative = 8;  // a negative length

// A step's new tokens: request i goes from lens[i] to lens[i] + new_lens[i] tokens.  The pages that takes come off the end of
// free_pages[0 .. *n_free), requests in order; token t of the batch (request i, cu_new[i] <= t < cu_new[i + 1]) has position
// positions[t] in its request and slot page * page_size + offset in the cache.  Rows behind the last token: slot -1, position 0.
void paged_extend(int* table, int* lens, const int* new_lens, const int* free_pages, int* n_free, int* cu_new, int64_t* slots, int* positions,
                  int* status, int requests, int width, int capacity, int page, int rows, cudaStream_t stream);
// The inverse: request i keeps its first keep_lens[i] tokens, pages that are not needed for them go back, table entries become -1.
void paged_trim(int* table, int* lens, const int* keep_lens, int* free_pages, int* n_free, int* status, int requests, int width, int capacity,
                int page, cudaStream_t stream);

// qkv: [rows, (hq + 2 hkv) * 128] at row_stride elements.  q_out [rows, hq * 128]: the queries, rotated by positions[t]; rotated keys and
// plain values of tokens with a slot in the cache go there (a slot that is negative or behind the cache: nowhere).
void rope_paged_append(DType t, const void* qkv, int64_t row_stride, void* q_out, void* kcache, void* vcache, const int64_t* slots,
                       const int* positions, int rows, int hq, int hkv, int page, int64_t pages, double theta, cudaStream_t stream);

struct PagedAttentionShape {
  int rows;        // of q and out
  int requests, hq, hkv;
  int page, width; // positions of a page, pages of a row of the block table
  int64_t pages;   // of the cache
  int max_new;     // no request has more new tokens
};
// What the first word of the attention's workspace says (bits) since it was zeroed.
constexpr int kPagedGaveUp = 1;   // a wait inside a kernel ran out: results are not valid, the workspace has to be zeroed
constexpr int kPagedMoreNew = 2;  // a request had more new tokens than max_new: its rows may not be written

// out[t] = softmax(q[t] k^T / sqrt(128)) v over the positions up to and including the token's own (0 where there are none); lens count the new
// tokens, cu_new starts with 0, rows behind its last are zeros.  A row that sees a score of NaN or +inf is NaN, and so is one all of whose
// scores are -inf, as softmax has it.  Behind a request's last position a page may hold anything, NaN included; an infinity or NaN among the
// values of a token may reach all rows of its request (0 x inf), as in any masked product.  Outputs are fp32 sums of weights of up to 2^8
// times values before they are divided: values of bf16 of 2^120 / positions and more may overflow there.
// The workspace is zero before the first call and kept between calls, which follow one another; it serves calls of every shape that it is
// large enough for.  `timeout_ns` bounds every wait inside the kernels; the longest is for an item of 256 rows in one span, some 17 ns a
// position (2 s for 10^8 of them).  Of the flags kMuteSends is known: one CTA leaves out its first copies, so the waits for these run out.
size_t paged_attention_workspace_bytes(int group, int max_new, int sm_count);
void paged_attention(DType t, const void* q, int64_t row_stride, const void* kcache, const void* vcache, const int* table, const int* lens,
                     const int* cu_new, void* out, void* workspace, const PagedAttentionShape& s, int sm_count, uint64_t timeout_ns, uint32_t flags, cudaStream_t stream);

struct VerifyShape {
  int requests, drafts;
  int64_t vocab;
  int64_t target_b, target_j, draft_b, draft_j;  // strides in elements
};
// Drafted tokens against the target's probabilities; draft, draft_lens nullptr: drafts without probabilities, all of them.
void verify_drafts(const float* target, const float* draft, const int64_t* tokens, const int* draft_lens, const float* accept, const float* sample,
                   int64_t* out, int* accepted, const VerifyShape& s, cudaStream_t stream);

}  // namespace b200ipc
