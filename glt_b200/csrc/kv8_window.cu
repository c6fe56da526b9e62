// glt_kv8_window_attention: a sliding window and a few first tokens (kv8_attention.cuh, Mode::kSinks).
//
// A sequence's steps of 32 tokens are those that hold its first tokens, and then those of its window; nothing between
// them is read, neither codes nor scales nor the block table.  Where the two meet they are one run.
#include "kv8_attention.cuh"

extern "C" int glt_kv8_window_attention(const GltKv8Cache* cache, const GltKv8Batch* batch, const uint16_t* q,
                                        int64_t ld_q, uint16_t* o, int64_t ld_o, float* lse, int num_heads,
                                        float scale, int window, int sinks, const uint8_t* token_mask,
                                        int64_t ld_mask, void* workspace, int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  if (sinks < 0) return glt::fail(GLT_EINVAL, "kv8: negative sinks");
  if (window == 0 || sinks == 0)   // without a window every token is visible as it is
    return glt_kv8_attention(cache, batch, q, ld_q, o, ld_o, lse, num_heads, scale, window, token_mask, ld_mask, workspace,
                             workspace_bytes, stream);
  if (batch->rows == 0 || batch->max_new == 0) return GLT_OK;
  glt::AttnArgs a;
  glt::Plan p;
  GLT_TRY(glt::prepare(cache, batch, q, ld_q, o, ld_o, lse, num_heads, scale, window, token_mask, ld_mask, workspace,
                       workspace_bytes, &a, &p));
  a.sinks = sinks;
  return glt::launch_all<glt::Mode::kSinks>(a, p, static_cast<cudaStream_t>(stream));
}
