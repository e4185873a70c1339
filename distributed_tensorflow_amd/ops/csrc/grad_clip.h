// Norm over all gradients of a model, and what is scaled by it (grad_clip.hip).
#pragma once
#include "common.h"

#include <vector>

struct ClipTensor {
  const void* in;
  void* out;          // null in a list that is only normed
  int64_t n;
  int dt;
};

// A list of tensors cut into launches: built once, holds addresses only.
class ClipList {
 public:
  explicit ClipList(const std::vector<ClipTensor>& tensors);
  // doubles of workspace that norm() fills and scale() reads
  size_t workspace_doubles() const { return partials_; }
  void norm(double* ws, hipStream_t s) const;                  // partial sums of squares
  void finish(const double* ws, float* norm, hipStream_t s) const;
  // out = in * min(1, clip / norm); the norm comes from `ws`, or from `use_norm` where that is given, and goes to `norm`
  void scale(const double* ws, const float* use_norm, float clip, float* norm, hipStream_t s) const;

  static constexpr int PER_LAUNCH = 128;
  struct Table {
    const void* in[PER_LAUNCH];
    void* out[PER_LAUNCH];
    int64_t n[PER_LAUNCH];            // elements, the element type in bits 60 and 61
    uint32_t first[PER_LAUNCH + 1];   // first chunk of each tensor
    int count;
  };

 private:
  struct Piece {
    Table table;
    int blocks;
    size_t at;        // its place in the workspace
  };
  std::vector<Piece> pieces_;
  size_t partials_ = 0;
};

int clipped_sgd_blocks(size_t n);
void launch_clipped_sgd_momentum_l2(float* p, const float* g, float* v, const float* l2x2, size_t n, float lr,
                                    float momentum, float grad_scale, float clip, const float* skip, double* ws,
                                    float* norm, hipStream_t s);
