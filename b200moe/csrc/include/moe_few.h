// Host interface of the few-token MoE layer (kernels/moe_few.cu).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace b200 {

constexpr int kFewMaxTokens = 64;
constexpr int kFewMaxExperts = 256;
constexpr int kFewMaxTopk = 8;

struct MoeFewArgs {
  const void* x;             // [T, H] bf16
  const void* router;        // [>= E, H] bf16
  const void* w13;           // [E, 2I, H] e4m3 (scales s13) or bf16
  const float* s13;          // [E, 2I / 128, H / 128]
  const void* w2;            // [E, H, I]
  const float* s2;           // [E, H / 128, I / 128]
  int fp8;
  int tiled;                 // e4m3 weights stored tile-major
  int T, H, I, E, topk, renorm;
  void* out;                 // [T, H] bf16
  int* ids;                  // [T, topk] chosen experts, may be null
  float* weights;            // [T, topk] their weights, may be null
  // workspace, 16-byte aligned
  float* logits;             // [T, E]
  void* x8;                  // e4m3 weights: [T, 2, H] e4m3, the two terms of x / x_factor
  float* x_factor;           // [T]
  void* h;                   // [T * topk, I] f16, h / h_factor (e4m3 weights), or [2, T * topk, I] bf16
  float* h_factor;           // [T * topk, I / 16]
  float* slots;              // [T * topk, H]
  int2* sel;                 // [T * topk] chosen experts and weights
  int* done;                 // [H / 128]
};
void moe_few(const MoeFewArgs& a, cudaStream_t s);

}  // namespace b200
