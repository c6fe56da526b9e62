// glt_kv8_attention: see kv8_attention.cuh for the kernels.
#include "kv8_attention.cuh"

extern "C" int glt_kv8_attention_workspace(const GltKv8Cache* cache, const GltKv8Batch* batch,
                                           int num_heads, int64_t* bytes) {
  if (!bytes) return glt::fail(GLT_EINVAL, "null argument");
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  *bytes = batch->rows > 0 && batch->max_new > 0 ? glt::plan(*cache, *batch, num_heads).bytes : 0;
  return GLT_OK;
}

extern "C" int glt_kv8_attention(const GltKv8Cache* cache, const GltKv8Batch* batch, const uint16_t* q,
                                 int64_t ld_q, uint16_t* o, int64_t ld_o, float* lse, int num_heads,
                                 float scale, int window, const uint8_t* token_mask, int64_t ld_mask,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  GLT_TRY(glt::check_heads(cache, batch, num_heads));
  if (batch->rows == 0 || batch->max_new == 0) return GLT_OK;
  glt::AttnArgs a;
  glt::Plan p;
  GLT_TRY(glt::prepare(cache, batch, q, ld_q, o, ld_o, lse, num_heads, scale, window, token_mask, ld_mask, workspace,
                       workspace_bytes, &a, &p));
  return glt::launch_all<glt::Mode::kPlain>(a, p, static_cast<cudaStream_t>(stream));
}
