// What host/q4t/model/verify_head.h refuses before it enqueues anything (no GPU needed: the addresses are never read).
// Prints "verify_refusals PASS" on success.
#include <cstdio>
#include <string>

#include "q4t/model/verify_head.h"

using namespace q4t;

int failures = 0;

template <typename T>
T* at(uintptr_t a) {
  return reinterpret_cast<T*>(a);
}

struct Step {
  uint16_t *x, *y;
  model::VerifyHeadWeights w;
  model::DraftBatch b;
  void* ws;
  size_t bytes;
};

Step good() {
  constexpr uintptr_t kM = uintptr_t{1} << 24;
  Step s{};
  s.x = at<uint16_t>(kM);
  s.y = at<uint16_t>(2 * kM);
  s.w.norm = at<uint16_t>(3 * kM);
  s.w.head = at<uint8_t>(4 * kM);
  s.w.head_scale = at<float>(5 * kM);
  s.w.hs = 256;
  s.w.vocab = 1001;
  s.b.B = 2;
  s.b.n = 3;
  s.b.draft_ids = at<int32_t>(6 * kM);
  s.b.draft_len = at<int32_t>(7 * kM);
  s.b.temperature = at<float>(8 * kM);
  s.b.uniforms = at<float>(9 * kM);
  s.b.draft_logits = at<uint16_t>(10 * kM);
  s.b.tokens = at<int32_t>(11 * kM);
  s.b.accepted = at<int32_t>(12 * kM);
  s.b.probs = at<float>(13 * kM);
  s.ws = at<void>(14 * kM);
  s.bytes = model::VerifyHeadWorkspaceBytes(2, 3, 256, 1001);
  return s;
}

template <typename F>
void refused(const char* text, F change) {
  Step s = good();
  change(s);
  const std::string got = model::VerifyHead(s.x, s.y, s.w, s.b, s.ws, s.bytes, nullptr).message();
  if (got.find(text) == std::string::npos) {
    std::printf("expected '%s', got '%s'\n", text, got.c_str());
    ++failures;
  }
}
template <typename T>
T* moved(T* p, int64_t bytes) {
  return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(p) + bytes);
}

int main() {
  // alignment, of what the norm itself does not see
  refused("16 bytes", [](Step& s) { s.w.head = moved(s.w.head, 8); });
  refused("aligned", [](Step& s) { s.w.head_scale = moved(s.w.head_scale, 2); });
  refused("aligned", [](Step& s) { s.b.draft_logits = moved(s.b.draft_logits, 1); });
  refused("4-byte", [](Step& s) { s.b.draft_ids = moved(s.b.draft_ids, 2); });
  refused("4-byte", [](Step& s) { s.b.draft_len = moved(s.b.draft_len, 1); });
  refused("4-byte", [](Step& s) { s.b.temperature = moved(s.b.temperature, 2); });
  refused("4-byte", [](Step& s) { s.b.uniforms = moved(s.b.uniforms, 2); });
  refused("4-byte", [](Step& s) { s.b.tokens = moved(s.b.tokens, 2); });
  refused("4-byte", [](Step& s) { s.b.accepted = moved(s.b.accepted, 3); });
  refused("4-byte", [](Step& s) { s.b.probs = moved(s.b.probs, 2); });
  refused("16 bytes", [](Step& s) { s.ws = moved(static_cast<uint8_t*>(s.ws), 8); });
  // outputs over inputs, within one call and across the step
  refused("tokens overlaps uniforms", [](Step& s) { s.b.tokens = at<int32_t>(reinterpret_cast<uintptr_t>(s.b.uniforms) + 28); });
  refused("accepted overlaps draft_ids", [](Step& s) { s.b.accepted = const_cast<int32_t*>(s.b.draft_ids); });
  refused("probs overlaps tokens", [](Step& s) { s.b.probs = at<float>(reinterpret_cast<uintptr_t>(s.b.tokens) + 4); });
  refused("x overlaps tokens", [](Step& s) { s.b.tokens = at<int32_t>(reinterpret_cast<uintptr_t>(s.x) + 8 * 256 * 2 - 4); });
  refused("head overlaps probs", [](Step& s) { s.b.probs = at<float>(reinterpret_cast<uintptr_t>(s.w.head)); });
  refused("x overlaps workspace", [](Step& s) { s.ws = moved(reinterpret_cast<uint8_t*>(s.x), 8 * 256 * 2 - 16); });
  refused("draft_logits overlaps workspace", [](Step& s) { s.b.draft_logits = at<uint16_t>(reinterpret_cast<uintptr_t>(s.ws) + 4096); });
  refused("norm overlaps workspace", [](Step& s) { s.w.norm = at<uint16_t>(reinterpret_cast<uintptr_t>(s.ws) + 8192); });
  refused("uniforms overlaps x", [](Step& s) { s.b.uniforms = at<float>(reinterpret_cast<uintptr_t>(s.x) + 64); });
  refused("head_scale overlaps x", [](Step& s) { s.w.head_scale = at<float>(reinterpret_cast<uintptr_t>(s.x)); });
  refused("y overlaps x", [](Step& s) { s.y = moved(s.x, 16); });
  // as before
  refused("null pointer", [](Step& s) { s.b.uniforms = nullptr; });
  refused("workspace too small", [](Step& s) { s.bytes -= 1; });
  refused("invalid dims", [](Step& s) { s.w.hs = 264; });
  if (failures) return 1;
  std::printf("verify_refusals PASS\n");
  return 0;
}
