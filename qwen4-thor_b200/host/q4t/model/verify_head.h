// The end of a decode step that verifies drafts (no counterpart in the reference's headers in this form): final norm with
// e4m3 output, head product, verification, on the C ABI.  The engine's ModelVerifyMulti hands the residual stream of
// B sequences x (1 target + n drafts) rows to VerifyHead and reads tokens and counts back.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <string>

#include "q4t/status.h"
#include "q4t_moe_b200.h"

namespace q4t::model {

// Head weights on the device: e4m3 rows with a scale each (q4t_quantize_rows_fp8 lays them out from bf16 once).
struct VerifyHeadWeights {
  const uint16_t* norm = nullptr;        // [hs] bf16, or null
  float norm_offset = 0.0f;              // 1 for a zero-centred norm weight
  float eps = 1e-6f;
  const uint8_t* head = nullptr;         // [vocab, hs] e4m3
  const float* head_scale = nullptr;     // [vocab]
  int hs = 0, vocab = 0;
};

// What is verified: B sequences with up to n drafts, rows as q4t_verify_args describes them.
struct DraftBatch {
  int B = 0, n = 0;
  const int32_t* draft_ids = nullptr;    // [B, n]
  const int32_t* draft_len = nullptr;    // [B] or null
  const float* temperature = nullptr;    // [B] or null
  const float* uniforms = nullptr;       // [B, n+1]
  const uint16_t* draft_logits = nullptr;  // [B*n, vocab] bf16 or null
  int32_t* tokens = nullptr;             // [B, n+1]
  int32_t* accepted = nullptr;           // [B]
  float* probs = nullptr;                // [B, n+1] or null
};

namespace detail {
struct VerifyHeadLayout {
  size_t codes, scales, logits, verify, total;
};
inline VerifyHeadLayout LayoutOf(int B, int n, int hs, int vocab) {
  auto up = [](size_t v) { return (v + 255) & ~size_t{255}; };
  const size_t rows = static_cast<size_t>(B) * (n + 1);
  VerifyHeadLayout L{};
  L.codes = 0;
  L.scales = up(rows * hs);
  L.logits = L.scales + up(rows * 4);
  L.verify = L.logits + up(rows * vocab * 2);
  L.total = L.verify + up(q4t_verify_drafts_workspace_bytes(B, n, vocab));
  return L;
}

// What the step writes (workspace, outputs, with y also x) lies over nothing else of the step.
inline Status Disjoint(const uint16_t* x, const uint16_t* y, const VerifyHeadWeights& w, const DraftBatch& b, const void* workspace,
                       size_t workspace_bytes) {
  struct Buffer {
    const char* name;
    const void* p;
    size_t bytes;
  };
  const size_t rows = static_cast<size_t>(b.B) * (b.n + 1), drafts = static_cast<size_t>(b.B) * b.n, hs = w.hs, vocab = w.vocab;
  const Buffer all[] = {{"workspace", workspace, workspace_bytes}, {"tokens", b.tokens, rows * 4}, {"accepted", b.accepted, b.B * size_t{4}},
                        {"probs", b.probs, rows * 4}, {"x", x, rows * hs * 2}, {"y", y, rows * hs * 2}, {"norm", w.norm, hs * 2},
                        {"head", w.head, vocab * hs}, {"head_scale", w.head_scale, vocab * 4}, {"draft_ids", b.draft_ids, drafts * 4},
                        {"draft_len", b.draft_len, b.B * size_t{4}}, {"temperature", b.temperature, b.B * size_t{4}},
                        {"uniforms", b.uniforms, rows * 4}, {"draft_logits", b.draft_logits, drafts * vocab * 2}};
  const int count = sizeof(all) / sizeof(all[0]), written = y ? 5 : 4;
  for (int i = 0; i < written; ++i)
    for (int j = i + 1; j < count; ++j) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(all[i].p), q = reinterpret_cast<uintptr_t>(all[j].p);
      if (p && q && p < q + all[j].bytes && q < p + all[i].bytes && !(all[i].p == x && all[j].p == y && x == y))
        return Status::Fail(std::string("verify head: ") + all[j].name + " overlaps " + all[i].name);
    }
  return Status();
}
}  // namespace detail

inline size_t VerifyHeadWorkspaceBytes(int B, int n, int hs, int vocab) {
  return q4t_verify_drafts_workspace_bytes(B, n, vocab) == 0 || hs <= 0 ? 0 : detail::LayoutOf(B, n, hs, vocab).total;
}

// x: residual stream bf16 [B*(n+1), hs], 16-byte aligned; y (may be null) is added to it first, in place.  Everything is
// enqueued on `stream`.  logits_out (may be null) receives the address of the bf16 logits in the workspace.  What is written (workspace,
// 16-byte aligned, outputs, with y also x) may not lie over anything else.  A refused call has changed nothing.
inline Status VerifyHead(uint16_t* x, const uint16_t* y, const VerifyHeadWeights& w, const DraftBatch& batch, void* workspace,
                         size_t workspace_bytes, cudaStream_t stream, const uint16_t** logits_out = nullptr) {
  const size_t need = VerifyHeadWorkspaceBytes(batch.B, batch.n, w.hs, w.vocab);
  if (need == 0 || w.hs % 16) return Status::Fail("verify head: invalid dims (hs must be a multiple of 16)");
  if (!x || !w.head || !batch.draft_ids || !batch.uniforms || !batch.tokens || !batch.accepted)   // before x changes
    return Status::Fail("verify head: null pointer");
  if (!workspace || workspace_bytes < need) return Status::Fail("workspace too small");
  const detail::VerifyHeadLayout L = detail::LayoutOf(batch.B, batch.n, w.hs, w.vocab);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(base + L.scales);
  uint16_t* logits = reinterpret_cast<uint16_t*>(base + L.logits);
  const int rows = batch.B * (batch.n + 1);
  q4t_linear_args l{};
  l.x = base + L.codes;
  l.w = w.head;
  l.M = rows;
  l.N = w.vocab;
  l.K = w.hs;
  l.fp8 = 1;
  l.x_scale = scales;
  l.w_scale = w.head_scale;
  l.out = logits;
  q4t_verify_args v{};
  v.target_logits = logits;
  v.draft_logits = batch.draft_logits;
  v.B = batch.B;
  v.n = batch.n;
  v.V = w.vocab;
  v.draft_ids = batch.draft_ids;
  v.draft_len = batch.draft_len;
  v.temperature = batch.temperature;
  v.uniforms = batch.uniforms;
  v.tokens = batch.tokens;
  v.accepted = batch.accepted;
  v.probs = batch.probs;
  // everything that is refused is refused before x changes: the later calls' arguments, and buffers of one call over another's
  const size_t verify_bytes = workspace_bytes - L.verify;
  if (q4t_linear_check(&l) != Q4T_OK || q4t_verify_drafts_check(&v, base + L.verify, verify_bytes) != Q4T_OK)
    return Status::Fail(q4t_last_error());
  if (Status s = detail::Disjoint(x, y, w, batch, workspace, need); !s.ok()) return s;
  if (q4t_residual_rmsnorm_fp8(x, y, y ? x : nullptr, w.norm, w.norm_offset, base + L.codes, scales, nullptr, rows, w.hs,
                               w.eps, stream) != Q4T_OK)
    return Status::Fail(q4t_last_error());
  if (q4t_linear(&l, stream) != Q4T_OK) return Status::Fail(q4t_last_error());
  if (q4t_verify_drafts(&v, base + L.verify, verify_bytes, stream) != Q4T_OK) return Status::Fail(q4t_last_error());
  if (logits_out) *logits_out = logits;
  return Status();
}

}  // namespace q4t::model
