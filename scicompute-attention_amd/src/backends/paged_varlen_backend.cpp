// Ragged chunks of new tokens over a paged KV cache: the host adapter of sca_hip_paged_varlen. Lengths
// come from the host (the cache's own, or the caller's), so the kernel library plans from them and
// nothing is uploaded.

#include <limits>
#include <string>
#include <vector>

#include "runtime/internal.hpp"
#include "scicompute_attention/capability.hpp"
#include "scicompute_attention/paged_attention.hpp"

namespace sca {
namespace {

sci::Result<AttentionResult> RunVarlen(const sci::Tensor& q, const PagedKVCache& kv,
                                       const PagedVarlenParams& params, const AttentionConfig& cfg) {
    auto fail = [](AttnStatusCode code, const std::string& msg) {
        return sci::MakeUnexpected<AttentionResult>(MakeStatus(code, "paged_attention_varlen " + msg));
    };
    if (q.ndims() != 3) {
        return fail(AttnStatusCode::kShapeMismatch,
                    "expects packed q=[T, H_q, D]; got ndims=" + std::to_string(q.ndims()));
    }
    const int64_t tokens = q.dim(0);
    const int64_t num_heads = q.dim(1);
    const int64_t head_dim = q.dim(2);
    const KVCacheConfig& kv_cfg = kv.Storage().Config();
    if (params.num_seqs < 1 || params.num_seqs > std::numeric_limits<int32_t>::max() / 2) {
        return fail(AttnStatusCode::kShapeMismatch, "num_seqs=" + std::to_string(params.num_seqs));
    }
    if (cfg.cu_seqlens_q == nullptr) {
        return fail(AttnStatusCode::kShapeMismatch, "requires host-resident cfg.cu_seqlens_q");
    }
    if (params.layer < 0 || params.layer >= kv_cfg.num_layers) {
        return fail(AttnStatusCode::kShapeMismatch, "layer=" + std::to_string(params.layer) +
                                                        " out of range [0," +
                                                        std::to_string(kv_cfg.num_layers) + ")");
    }
    if (q.dtype() != sci::DType::kFloat16 && q.dtype() != sci::DType::kBFloat16) {
        return fail(AttnStatusCode::kUnsupportedDtype,
                    std::string("computes in fp16/bf16; dtype=") + sci::kDTypeName(q.dtype()));
    }
    if (q.dtype() != kv_cfg.dtype) {
        return fail(AttnStatusCode::kUnsupportedDtype,
                    std::string("dtype mismatch: q=") + sci::kDTypeName(q.dtype()) +
                        ", cache=" + sci::kDTypeName(kv_cfg.dtype));
    }
    if (head_dim != kv_cfg.head_dim) {
        return fail(AttnStatusCode::kShapeMismatch,
                    "head_dim=" + std::to_string(head_dim) + " differs from the cache's head_dim=" +
                        std::to_string(kv_cfg.head_dim));
    }
    if (num_heads < kv_cfg.num_kv_heads || num_heads % kv_cfg.num_kv_heads != 0) {
        return fail(AttnStatusCode::kShapeMismatch,
                    "num_heads=" + std::to_string(num_heads) +
                        " is not a multiple of the cache's num_kv_heads=" +
                        std::to_string(kv_cfg.num_kv_heads));
    }
    if (cfg.sliding_window > 0) {
        return fail(AttnStatusCode::kUnsupportedFeature,
                    "sliding_window=" + std::to_string(cfg.sliding_window) + " not implemented");
    }
    if (cfg.softcap > 0.0f) {
        return fail(AttnStatusCode::kUnsupportedFeature,
                    "softcap=" + std::to_string(cfg.softcap) + " not implemented");
    }
    if (q.device_type() != sci::DeviceType::kGPU) {
        return fail(AttnStatusCode::kUnsupportedFeature, "requires a GPU query");
    }
    const int32_t* page_table = params.page_table != nullptr ? params.page_table : kv.PageTableDevicePtr();
    if (page_table == nullptr || kv.Storage().K(params.layer).device_type() != sci::DeviceType::kGPU ||
        kv.Storage().K(params.layer).device().id() != q.device().id()) {
        return fail(AttnStatusCode::kShapeMismatch, "needs q and the cache on one GPU");
    }
    if (params.page_table != nullptr && (params.kv_lens == nullptr || params.max_blocks_per_seq < 1)) {
        return fail(AttnStatusCode::kShapeMismatch,
                    "with a page table of the caller's needs kv_lens and max_blocks_per_seq");
    }

    // Sequences: rows of the page table, lengths, and the packed tokens they own.
    const size_t n = static_cast<size_t>(params.num_seqs);
    std::vector<int32_t> rows(n), lens(n);
    if (cfg.cu_seqlens_q[0] != 0) {
        return fail(AttnStatusCode::kShapeMismatch,
                    "cu_seqlens_q starts at " + std::to_string(cfg.cu_seqlens_q[0]) + ", not 0");
    }
    for (size_t s = 0; s < n; ++s) {
        const int64_t id = params.seq_ids != nullptr ? params.seq_ids[s] : static_cast<int64_t>(s);
        const int64_t most = params.page_table != nullptr ? std::numeric_limits<int32_t>::max() : kv.MaxNumSeqs();
        if (id < 0 || id >= most) {
            return fail(AttnStatusCode::kShapeMismatch, "sequence id " + std::to_string(id) +
                                                            " out of range [0," + std::to_string(most) + ")");
        }
        const int64_t len = params.kv_lens != nullptr ? params.kv_lens[s] : kv.SeqLength(id);
        if (len < 0) {
            return fail(AttnStatusCode::kShapeMismatch,
                        "kv_lens[" + std::to_string(s) + "]=" + std::to_string(len));
        }
        if (len > std::numeric_limits<int32_t>::max()) {
            return fail(AttnStatusCode::kSeqTooLong, "sequence " + std::to_string(id) + " has " +
                                                         std::to_string(len) + " keys");
        }
        if (cfg.cu_seqlens_q[s + 1] < cfg.cu_seqlens_q[s] || cfg.cu_seqlens_q[s + 1] > tokens) {
            return fail(AttnStatusCode::kShapeMismatch,
                        "cu_seqlens_q[" + std::to_string(s + 1) + "]=" +
                            std::to_string(cfg.cu_seqlens_q[s + 1]) + " decreases or passes T=" +
                            std::to_string(tokens));
        }
        rows[s] = static_cast<int32_t>(id);
        lens[s] = static_cast<int32_t>(len);
    }

    AttentionResult result;
    result.out = sci::Tensor(sci::TensorShape({tokens, num_heads, head_dim}), q.dtype(), q.device());
    if (result.out.data() == nullptr && tokens > 0) {
        return fail(AttnStatusCode::kWorkspaceExceeded, "allocation of the output failed");
    }
    if (cfg.return_lse) {
        result.lse = sci::Tensor(sci::TensorShape({tokens, num_heads}), sci::DType::kFloat32, q.device());
        if (result.lse.data() == nullptr && tokens > 0) {
            return fail(AttnStatusCode::kWorkspaceExceeded, "allocation of the LSE buffer failed");
        }
    }
    AttentionShape shape;
    shape.head_dim = head_dim;
    const int64_t q_token = num_heads * head_dim;
    const int64_t kv_token = kv_cfg.num_kv_heads * head_dim;
    sca_paged_varlen_params p{};
    p.q = q.data();
    p.k = kv.Storage().K(params.layer).data();
    p.v = kv.Storage().V(params.layer).data();
    p.k_exp = static_cast<const uint8_t*>(kv.Storage().KExponents(params.layer).data());
    p.v_exp = static_cast<const uint8_t*>(kv.Storage().VExponents(params.layer).data());
    p.out = result.out.data();
    p.lse = cfg.return_lse ? static_cast<float*>(result.lse.data()) : nullptr;
    p.page_table = page_table;
    p.cu_seqlens_q = cfg.cu_seqlens_q;
    p.kv_lens = lens.data();
    p.table_rows = rows.data();
    p.num_seqs = params.num_seqs;
    p.num_heads = num_heads;
    p.num_kv_heads = kv_cfg.num_kv_heads;
    p.head_dim = head_dim;
    p.block_size = kv.BlockSize();
    p.max_blocks_per_seq = params.page_table != nullptr ? params.max_blocks_per_seq : kv.MaxBlocksPerSeq();
    p.num_kv_blocks = kv_cfg.num_blocks;
    p.q_ss = q_token, p.q_sh = head_dim;
    p.k_ss = kv_token, p.k_sh = head_dim;
    p.v_ss = kv_token, p.v_sh = head_dim;
    p.o_ss = q_token, p.o_sh = head_dim;
    p.scale = EffectiveScale(cfg, shape);
    p.causal = cfg.causal ? 1 : 0;
    p.dtype = runtime::KernelDtype(q.dtype());

    void* stream = runtime::StreamHandle(cfg.stream);
    // Tokens behind the last sequence (a padded batch): zeros.
    const int64_t used = cfg.cu_seqlens_q[n];
    sci::Status status = sci::Status::Ok();
    if (used < tokens) {
        const int64_t eb = DtypeSize(q.dtype());
        status = runtime::StatusFromHip(
            sca_hip_zero_async(static_cast<char*>(result.out.data()) + used * q_token * eb,
                               static_cast<size_t>((tokens - used) * q_token * eb), stream),
            "paged varlen padding");
        if (status.ok() && cfg.return_lse) {
            status = runtime::StatusFromHip(
                sca_hip_zero_async(static_cast<float*>(result.lse.data()) + used * num_heads,
                                   static_cast<size_t>((tokens - used) * num_heads) * sizeof(float), stream),
                "paged varlen padding");
        }
        if (!status.ok()) return sci::MakeUnexpected<AttentionResult>(status);
    }
    int64_t bytes = 0;
    if (used > 0) {
        if (cfg.num_splits != 1) bytes = sca_hip_paged_varlen_bytes(&p);
        const int64_t limit = static_cast<int64_t>(cfg.workspace_limit_bytes);
        if (limit > 0 && bytes > limit) bytes = limit;
        // States of a run that splits its keys (most need none; without scratch it runs unsplit).
        const runtime::StreamScratch scratch(static_cast<size_t>(bytes), q.device().id(), stream);
        if (scratch.ptr == nullptr) bytes = 0;
        status = runtime::StatusFromHip(sca_hip_paged_varlen(&p, scratch.ptr, bytes, stream), "paged varlen");
        if (!status.ok()) return sci::MakeUnexpected<AttentionResult>(status);
    }
    result.stats.used_backend = BackendKind::kPaged;
    result.stats.workspace_bytes = static_cast<size_t>(bytes);
    result.stats.kv_bytes = kv.Storage().MemoryBytes();
    result.stats.note = "paged varlen: " + std::to_string(used) + " new tokens of " +
                        std::to_string(params.num_seqs) + " sequences, block_size=" +
                        std::to_string(kv.BlockSize()) + ", layer=" + std::to_string(params.layer) +
                        (p.k_exp != nullptr ? ", 8-bit pages" : "");
    return sci::Ok(std::move(result));
}

}  // namespace

sci::Result<AttentionResult> paged_attention_varlen(const sci::Tensor& q, const PagedKVCache& kv,
                                                    const PagedVarlenParams& params,
                                                    const AttentionConfig& cfg) {
    return RunVarlen(q, kv, params, cfg);
}

}  // namespace sca
