// Norm over all gradients of a model, and what is scaled by it (grad_clip.hip).
#pragma once
#include "common.h"

#include <string>
#include <vector>

struct ClipEntry {
  const void* in;
  void* out;            // null in a list that is only normed
  int64_t bytes;
  uint32_t first;       // its first chunk
  int32_t dt;
};

// A list of tensors cut into chunks, built once; it holds addresses only.  Walked either from tables in the kernels'
// arguments, PER_LAUNCH tensors a launch, or from a table in device memory in one launch (`resident`).
class ClipList {
 public:
  ClipList(const std::vector<uintptr_t>& in, const std::vector<uintptr_t>& out, const std::vector<int64_t>& n,
           const std::vector<int>& dt);
  // What `resident` has to point to: the entries, then a chunk's entry for every chunk.  Empty: one launch does anyway.
  std::string table() const;
  size_t pieces() const { return pieces_.size(); }      // launches of a sweep without `resident`
  size_t workspace_doubles() const { return partials_; }
  void norm(const void* resident, double* ws, hipStream_t s) const;                  // partial sums of squares
  void finish(const void* resident, const double* ws, float* norm, hipStream_t s) const;
  // out = in * min(1, clip / norm); the norm comes from `ws`, or from `use_norm` where that is given, and goes to `norm`
  void scale(const void* resident, double* ws, const float* use_norm, float clip, float* norm, hipStream_t s) const;

  static constexpr int PER_LAUNCH = 120;
  struct Table {        // a kernel argument: under 4 KB
    ClipEntry e[PER_LAUNCH];
    int count;
    uint32_t chunks;
  };

 private:
  int partials(const void* resident) const;
  struct Piece {
    Table table;
    size_t at;          // its place in the workspace
  };
  std::vector<ClipEntry> all_;      // `first` counts through the whole list
  uint64_t chunks_ = 0;
  std::vector<Piece> pieces_;
  size_t partials_ = 0;
  int64_t bytes_ = 0;
  bool in_place_ = true, outputs_ = true;
};

int clipped_sgd_blocks(size_t n);
void launch_clipped_sgd_momentum_l2(float* p, const float* g, float* v, const float* l2x2, size_t n, float lr,
                                    float momentum, float grad_scale, float clip, const float* skip, double* ws,
                                    float* norm, hipStream_t s);
