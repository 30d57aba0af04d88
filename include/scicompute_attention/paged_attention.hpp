#pragma once

#include <cstdint>

#include "scicompute_attention/attention_config.hpp"
#include "scicompute_attention/attention_result.hpp"
#include "scicompute_attention/export.hpp"
#include "scicompute_attention/paged_kv_cache.hpp"

namespace sca {

struct PagedAttentionParams {
    const int32_t* page_table{nullptr};  // device [num_seqs, max_blocks_per_seq]; null => kv's own
    const int32_t* seq_lens{nullptr};    // device [num_seqs] (including the new token); null =>
                                         // every mapped page of the row is attended in full
    int64_t num_seqs{0};
    int64_t block_size{16};
    int64_t max_blocks_per_seq{0};       // 0 => kv.MaxBlocksPerSeq()
    int64_t layer{0};                    // which KV layer to read
};

// Decode over a paged KV cache: q is [num_seqs, H_q, 1, D] BHSD. A cache with 8-bit storage is attended
// as the values its codes stand for (params.block_size must then be the cache's own).
SCI_ATTENTION_API sci::Result<AttentionResult> paged_attention(const sci::Tensor& q,
                                                               const PagedKVCache& kv,
                                                               const PagedAttentionParams& params,
                                                               const AttentionConfig& cfg);

SCI_ATTENTION_API sci::Result<AttentionResult> paged_attention(const sci::Tensor& q,
                                                               const PagedKVCache& kv,
                                                               const AttentionConfig& cfg);

// Ragged chunks of new tokens over a paged KV cache (no counterpart in the reference, whose paged path
// takes one query token per sequence): prompts, parts of prompts, drafted tokens and single tokens in
// one call. Everything here lives on the host but page_table.
struct PagedVarlenParams {
    const int64_t* seq_ids{nullptr};     // host [num_seqs]: the cache's sequences, in the order of the
                                         // packed tokens; null => 0, 1, ... (an id may repeat)
    const int32_t* kv_lens{nullptr};     // host [num_seqs]: keys to attend, the new tokens' included;
                                         // null => the cache's lengths
    int64_t num_seqs{0};
    int64_t layer{0};                    // which KV layer to read
    const int32_t* page_table{nullptr};  // device [rows, max_blocks_per_seq], row seq_ids[s]; null =>
                                         // kv's own. With a table of the caller's, kv_lens is needed.
    int64_t max_blocks_per_seq{0};       // of that table
};

// q is packed [T, H_q, D] (fp16 or bf16) and cfg.cu_seqlens_q (host, num_seqs + 1, from 0, not
// decreasing) says which tokens are whose: sequence s's new tokens are the last of its keys, which the
// cache already holds (append first, then attend). Returns out [T, H_q, D] and, with cfg.return_lse, an
// FP32 lse [T, H_q]. With cfg.causal new token i of n sees keys j <= i + kv_len - n, else every key. A
// token that sees no key (none mapped, kv_len 0) gives zeros and an lse of -inf; tokens behind the last
// sequence give zeros. cfg.num_splits = 1 keeps every row tile's keys in one workgroup (no workspace);
// other values leave the split to the plan, as far as cfg.workspace_limit_bytes allows.
SCI_ATTENTION_API sci::Result<AttentionResult> paged_attention_varlen(const sci::Tensor& q,
                                                                      const PagedKVCache& kv,
                                                                      const PagedVarlenParams& params,
                                                                      const AttentionConfig& cfg);

}  // namespace sca
