// MXFP4 experts: what the layer call and the two files of kernels share.
#pragma once

#include "common.h"

namespace wisp {

// How a call is computed (mxfp4_plan): in the two launches for a few tokens, or
// by the grouped GEMM with w2's k range in `splits` parts.
struct Mxfp4Plan {
  bool few;
  int splits;
};
Mxfp4Plan mxfp4_plan(int T, int K, int H, int I, int experts);
size_t mxfp4_work_bytes(const Mxfp4Plan& plan, int T, int K, int H, int I, int nslots);
const char* mxfp4_unsupported(int H, int I, int K);

// SwiGLU experts of (part of) a call; strides in bytes.
int experts_mxfp4(const Mxfp4Plan& plan, const void* x, int T, int H, int I, int K,
                  const float* topk_w, const int32_t* slots, int nslots, const void* w13,
                  size_t w13_stride, const void* s13, size_t s13_stride, const void* w2,
                  size_t w2_stride, const void* s2, size_t s2_stride, void* act, void* out,
                  void* work, size_t work_bytes, hipStream_t st, const StageEvents* ev);
int layer_mxfp4(const Mxfp4Plan& plan, const void* x, const void* logits, int logits_dtype,
                int renorm, int64_t* forward, int T, int H, int I, int K, float* topk_w,
                int32_t* ids, int experts, const void* w13, size_t w13_stride, const void* s13,
                size_t s13_stride, const void* w2, size_t w2_stride, const void* s2,
                size_t s2_stride, void* act, void* out, void* work, size_t work_bytes,
                hipStream_t st, const StageEvents* ev);

// The two launches: whether they serve a call, the bytes between them, and
// they themselves.  With logits they route (and write topk_w and slots), else
// topk_w and slots are the caller's.
bool mxfp4_few(int T, int K, int H, int I, int nslots);
size_t mxfp4_few_bytes(int P, int I);
int mxfp4_few_layer(const void* x, const void* logits, int logits_dtype, int renorm,
                    int64_t* forward, int T, int H, int I, int K, float* topk_w, int32_t* slots,
                    int nslots, const void* w13, size_t w13_stride, const void* s13,
                    size_t s13_stride, const void* w2, size_t w2_stride, const void* s2,
                    size_t s2_stride, void* act, void* out, hipStream_t st, const StageEvents* ev);

}  // namespace wisp
