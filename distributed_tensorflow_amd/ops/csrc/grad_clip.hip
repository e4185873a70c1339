// Global gradient norm, clipping to it, and the momentum update with the clipped gradient.
//
//   norm = sqrt(sum over all tensors of g^2)      out = g * min(1, clip / norm)
//
// Two launches: the first leaves a partial sum per block, in the second every block adds the up to 1024 partial
// sums itself (in a fixed order, so a third launch, a ticket and atomics are not needed and the bits are the same
// every time) and scales.  A list that takes several launches has its partial sums added by one in between.  Both are
// sweeps bound by memory; the second walks from the end, where the first has left the memory-side cache filled.
//
// Squares are taken and summed in 64 bits: they cannot overflow or vanish for any fp32 or bf16 gradient, and a sum
// of hundreds of millions keeps its digits; the sweeps are bound by memory all the same.
//
// A norm that is infinite or NaN makes every result NaN, as TensorFlow's clip_by_global_norm has it; a norm of zero
// leaves the gradients alone.
//
// Tensors are cut into chunks of 8 KB that never cross a tensor; the blocks walk the chunks side by side, four blocks a CU
// (a narrow front over the memory; 400 M mixed elements: 419 us, chunks of 16 KB 436, of 4 KB 545; with runs of chunks of
// each block's own 538).  Which tensor a chunk belongs to is looked up while the chunk before it is loaded: in a table in the
// kernel's arguments (a list given as such: nothing to upload and keep alive, and a captured launch holds its own copy), or
// in device memory (a table that is kept: any number of tensors in one launch).
//
// Measured: 161 tensors of 25.6 M fp32 elements 18 + 34 us (5.7 and 6.0 TB/s), 384 of 400 M mixed ones 122 + 293 us (6.6 and
// 5.5 TB/s); what bounds both is memory, and that the norm has to be known before the first element can be scaled.
#include <algorithm>
#include <stdexcept>

#include "grad_clip.h"

namespace {

constexpr int TPB = 256;
constexpr int U = 2;          // accesses of 16 bytes a thread and chunk
constexpr int CHUNK_BYTES = TPB * 16 * U;
constexpr int MAX_BLOCKS = 1024;                   // per launch: four a CU
constexpr int FOLD_TPB = 1024;
constexpr int SGD_BLOCKS = 512;                    // of the update's two sweeps
constexpr int64_t CACHE_BYTES = 192 << 20;         // of what a sweep leaves in the memory-side cache (256 MB)

typedef u32x4 __attribute__((aligned(2))) Any16;   // any address will do

template <int DT>
__device__ __forceinline__ int unpack(const u32x4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == DT_F32) {
      f[j] = __uint_as_float(w[j]);
    } else {
      f[2 * j] = lo16<DT>(w[j]);
      f[2 * j + 1] = hi16<DT>(w[j]);
    }
  }
  return DT == DT_F32 ? 4 : 8;
}
template <int DT>
__device__ __forceinline__ u32x4 scaled(const u32x4 v, float factor) {
  float f[8];
  unpack<DT>(v, f);
  u32x4 o;
  if constexpr (DT == DT_F32) {
    o.x = __float_as_uint(f[0] * factor); o.y = __float_as_uint(f[1] * factor);
    o.z = __float_as_uint(f[2] * factor); o.w = __float_as_uint(f[3] * factor);
  } else {
    o.x = pack2<DT>(f[0] * factor, f[1] * factor); o.y = pack2<DT>(f[2] * factor, f[3] * factor);
    o.z = pack2<DT>(f[4] * factor, f[5] * factor); o.w = pack2<DT>(f[6] * factor, f[7] * factor);
  }
  return o;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ double block_sum64(double v, double* red) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0] + red[1] + red[2] + red[3];
  __syncthreads();
  return v;
}

// min(1, clip / norm) of the partial sums (or of a norm that is given), the same value in every thread.
__device__ __forceinline__ float clip_factor(const double* ws, int partials, const float* use_norm, float clip,
                                             float* norm_out, double* red) {
  double norm;
  if (use_norm) {
    norm = (double)use_norm[0];
  } else {
    double s = 0.;
    for (int i = threadIdx.x; i < partials; i += TPB) s += ws[i];
    norm = sqrt(block_sum64(s, red));
  }
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
  if (!(norm < (double)INFINITY)) return __builtin_nanf("");
  return norm > (double)clip ? (float)((double)clip / norm) : 1.f;
}

struct Inline {         // a table in the arguments
  ClipList::Table t;
  __device__ __forceinline__ uint32_t chunks() const { return t.chunks; }
  __device__ __forceinline__ ClipEntry at(uint32_t c) const {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.e[mid].first <= c) lo = mid; else hi = mid - 1;
    }
    return t.e[lo];
  }
};
struct Resident {       // a table in device memory
  const ClipEntry* e;
  const uint32_t* map;
  uint32_t n;
  __device__ __forceinline__ uint32_t chunks() const { return n; }
  __device__ __forceinline__ ClipEntry at(uint32_t c) const { return e[map[c]]; }
};

// A thread's pieces of 16 bytes of a chunk; past the tensor's end: zeros.
template <bool NT>
__device__ __forceinline__ void load_chunk(const ClipEntry& e, uint32_t c, u32x4* v) {
  const int64_t at = (int64_t)(c - e.first) * CHUNK_BYTES + (int64_t)threadIdx.x * 16;
  const char* p = reinterpret_cast<const char*>(e.in);
  if (at - (int64_t)threadIdx.x * 16 + CHUNK_BYTES <= e.bytes) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Any16* q = reinterpret_cast<const Any16*>(p + at + k * TPB * 16);
      if constexpr (NT) v[k] = __builtin_nontemporal_load(q);
      else v[k] = *q;
    }
  } else {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t o = at + k * TPB * 16;
      v[k] = u32x4{0u, 0u, 0u, 0u};
      if (o + 16 <= e.bytes) {
        v[k] = *reinterpret_cast<const Any16*>(p + o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (o + 2 * j < e.bytes) v[k][j >> 1] |= (uint32_t)*reinterpret_cast<const uint16_t*>(p + o + 2 * j) << (16 * (j & 1));
      }
    }
  }
}

template <bool NT>
__device__ __forceinline__ void store_chunk(const ClipEntry& e, uint32_t c, const u32x4* v) {
  const int64_t at = (int64_t)(c - e.first) * CHUNK_BYTES + (int64_t)threadIdx.x * 16;
  char* p = reinterpret_cast<char*>(e.out);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int64_t o = at + k * TPB * 16;
    if (o + 16 <= e.bytes) {
      Any16* q = reinterpret_cast<Any16*>(p + o);
      if constexpr (NT) __builtin_nontemporal_store((Any16)v[k], q);
      else *q = v[k];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (o + 2 * j < e.bytes) *reinterpret_cast<uint16_t*>(p + o + 2 * j) = (uint16_t)(v[k][j >> 1] >> (16 * (j & 1)));
    }
  }
}

template <int DT>
__device__ __forceinline__ void add_squares(const u32x4* v, double* s) {
#pragma unroll
  for (int k = 0; k < U; ++k) {
    float f[8];
    const int n = unpack<DT>(v[k], f);
#pragma unroll
    for (int j = 0; j < n; ++j) s[j & 3] = fma((double)f[j], (double)f[j], s[j & 3]);
  }
}

// Chunks before `cold` go past the caches: the sweep leaves the list's end there, where the scaling begins.
template <typename T>
__global__ __launch_bounds__(TPB) void norm_kernel(const T t, uint32_t cold, double* __restrict__ ws) {
  __shared__ double red[4];
  double s[4] = {0., 0., 0., 0.};
  const uint32_t chunks = t.chunks();
  uint32_t c = blockIdx.x;
  ClipEntry e = {};
  if (c < chunks) e = t.at(c);
  while (c < chunks) {
    u32x4 v[U];
    if (c < cold) load_chunk<true>(e, c, v);
    else load_chunk<false>(e, c, v);
    const int dt = e.dt;
    c += gridDim.x;
    if (c < chunks) e = t.at(c);
    switch (dt) {
      case DT_BF16: add_squares<DT_BF16>(v, s); break;
      case DT_F16: add_squares<DT_F16>(v, s); break;
      default: add_squares<DT_F32>(v, s); break;
    }
  }
  const double sum = block_sum64((s[0] + s[1]) + (s[2] + s[3]), red);
  if (threadIdx.x == 0) ws[blockIdx.x] = sum;
}

__global__ __launch_bounds__(TPB) void norm_finish_kernel(const double* __restrict__ ws, int partials, float* norm) {
  __shared__ double red[4];
  (void)clip_factor(ws, partials, nullptr, 1.f, norm, red);
}

// One block adds the partial sums of several launches to the first of them.  Without it every block of every launch of the
// scaling adds all of them, which is quadratic in the launches: 3600 tensors of 100 000 floats in 30 launches 1418 us of
// scaling, 628 with this; two launches (161 tensors) 44.1 and 43.4.
__global__ __launch_bounds__(FOLD_TPB) void fold_kernel(double* __restrict__ ws, int partials) {
  __shared__ double red[FOLD_TPB / 64];
  double s = 0.;
#pragma unroll 8
  for (int i = threadIdx.x; i < partials; i += FOLD_TPB) s += ws[i];
  s = wave_sum64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();                      // every partial sum has been read
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < FOLD_TPB / 64; ++w) s += red[w];
    ws[0] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(TPB) void scale_kernel(const T t, const double* __restrict__ ws, int partials,
                                                    const float* __restrict__ use_norm, float clip, float* norm,
                                                    int in_place, int nt) {
  __shared__ double red[4];
  const float factor = clip_factor(ws, partials, use_norm, clip, norm, red);
  if (in_place && factor == 1.f) return;        // every result is where it belongs already
  const uint32_t chunks = t.chunks();
  uint32_t k = blockIdx.x;                      // from the end, which the norm's sweep has left in the cache
  ClipEntry next = {};
  if (k < chunks) next = t.at(chunks - 1 - k);
  while (k < chunks) {
    const ClipEntry e = next;
    const uint32_t c = chunks - 1 - k;
    u32x4 v[U];
    load_chunk<false>(e, c, v);
    k += gridDim.x;
    if (k < chunks) next = t.at(chunks - 1 - k);
#pragma unroll
    for (int i = 0; i < U; ++i)
      v[i] = e.dt == DT_BF16 ? scaled<DT_BF16>(v[i], factor) : e.dt == DT_F16 ? scaled<DT_F16>(v[i], factor)
                                                                               : scaled<DT_F32>(v[i], factor);
    if (nt) store_chunk<true>(e, c, v);
    else store_chunk<false>(e, c, v);
  }
}

// ---- the update ---------------------------------------------------------------------------------
//   g' = g * grad_scale + l2x2 * w      f = min(1, clip / |g'|)      v = momentum v - lr f g'      w += v
// (the norm is that of the whole gradient, the regulariser's part included, as an optimizer sees it)
// Three streams are read for the norm, four read and two written for the update; both run best as a narrow front with
// one access of a kind under way a thread and 512 blocks (25.6 M elements: 157 us; with four 165, 1024 blocks 177).

__device__ __forceinline__ void unscale(const float* skip, float* grad_scale) {
  if (skip) *grad_scale *= skip[1];
}

__global__ __launch_bounds__(TPB) void sgd_norm_kernel(const float* __restrict__ p, const float* __restrict__ g,
                                                       const float* __restrict__ l2x2, size_t n, float grad_scale,
                                                       const float* __restrict__ skip, size_t cold, double* __restrict__ ws) {
  __shared__ double red[4];
  unscale(skip, &grad_scale);
  const size_t n4 = n / 4, stride = (size_t)gridDim.x * TPB;
  double s[4] = {0., 0., 0., 0.};
  auto take = [&](const f32x4 w, const f32x4 gr, const f32x4 l2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double d = (double)(gr[j] * grad_scale + l2[j] * w[j]);
      s[j] = fma(d, d, s[j]);
    }
  };
  for (size_t i = blockIdx.x * (size_t)TPB + threadIdx.x; i < n4; i += stride) {
    const f32x4 *pw = reinterpret_cast<const f32x4*>(p) + i, *pg = reinterpret_cast<const f32x4*>(g) + i;
    const f32x4* pl = reinterpret_cast<const f32x4*>(l2x2) + i;
    if (i < cold) take(__builtin_nontemporal_load(pw), __builtin_nontemporal_load(pg), __builtin_nontemporal_load(pl));
    else take(*pw, *pg, *pl);
  }
  const size_t t = n4 * 4 + threadIdx.x;
  if (blockIdx.x == 0 && t < n) {
    const double d = (double)(g[t] * grad_scale + l2x2[t] * p[t]);
    s[0] = fma(d, d, s[0]);
  }
  const double sum = block_sum64((s[0] + s[1]) + (s[2] + s[3]), red);
  if (threadIdx.x == 0) ws[blockIdx.x] = sum;
}

template <bool NT>
__device__ __forceinline__ void update(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ v,
                                       const float* __restrict__ l2x2, size_t i, float momentum, float grad_scale,
                                       float step) {
  f32x4 w = reinterpret_cast<const f32x4*>(p)[i];
  const f32x4 gr = reinterpret_cast<const f32x4*>(g)[i], l2 = reinterpret_cast<const f32x4*>(l2x2)[i];
  const f32x4 d = gr * grad_scale + l2 * w;
  if (momentum != 0.f) {
    f32x4* pv = reinterpret_cast<f32x4*>(v) + i;
    f32x4 vel = NT ? __builtin_nontemporal_load(pv) : *pv;
    vel = vel * momentum - d * step;
    w += vel;
    if constexpr (NT) __builtin_nontemporal_store(vel, pv);
    else *pv = vel;
  } else {
    w -= d * step;
  }
  if constexpr (NT) __builtin_nontemporal_store(w, reinterpret_cast<f32x4*>(p) + i);
  else reinterpret_cast<f32x4*>(p)[i] = w;
}

__global__ __launch_bounds__(TPB) void clipped_sgd_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                          float* __restrict__ v, const float* __restrict__ l2x2,
                                                          size_t n, float lr, float momentum, float grad_scale,
                                                          float clip, const float* __restrict__ skip,
                                                          const double* __restrict__ ws, int partials, float* norm,
                                                          int nt) {
  __shared__ double red[4];
  unscale(skip, &grad_scale);
  const float factor = clip_factor(ws, partials, nullptr, clip, norm, red);
  if (skip && skip[0] != 0.f) return;       // a gradient is not finite: the step is left out
  const float step = lr * factor;
  const size_t n4 = n / 4, stride = (size_t)gridDim.x * TPB;
  if (blockIdx.x == 0 && n4 * 4 + threadIdx.x < n) {
    const size_t t = n4 * 4 + threadIdx.x;
    const float w = p[t], d = g[t] * grad_scale + l2x2[t] * w;
    float vel = -(d * step);
    if (momentum != 0.f) { vel = v[t] * momentum - d * step; v[t] = vel; }
    p[t] = w + vel;
  }
  // from the end, which the norm's sweep has left in the cache
  const size_t first = blockIdx.x * (size_t)TPB + threadIdx.x;
  if (nt) {
    for (size_t k = first; k < n4; k += stride) update<true>(p, g, v, l2x2, n4 - 1 - k, momentum, grad_scale, step);
  } else {
    for (size_t k = first; k < n4; k += stride) update<false>(p, g, v, l2x2, n4 - 1 - k, momentum, grad_scale, step);
  }
}

int elem_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }

}  // namespace

ClipList::ClipList(const std::vector<uintptr_t>& in, const std::vector<uintptr_t>& out, const std::vector<int64_t>& n,
                   const std::vector<int>& dt) {
  if (n.size() != in.size() || dt.size() != in.size() || (!out.empty() && out.size() != in.size()))
    throw std::invalid_argument("ClipList: lists of different lengths");
  for (size_t i = 0; i < in.size(); ++i) {
    if (dt[i] != DT_BF16 && dt[i] != DT_F16 && dt[i] != DT_F32) throw std::invalid_argument("unknown element type");
    if (n[i] < 0 || n[i] >= (1ll << 40)) throw std::invalid_argument("a tensor of up to 2^40 elements");
    if (n[i] == 0) continue;
    ClipEntry e;
    e.in = reinterpret_cast<const void*>(in[i]);
    e.out = out.empty() ? nullptr : reinterpret_cast<void*>(out[i]);
    e.bytes = n[i] * elem_bytes(dt[i]);
    e.dt = dt[i];
    e.first = (uint32_t)chunks_;
    chunks_ += ((uint64_t)e.bytes + CHUNK_BYTES - 1) / CHUNK_BYTES;
    if (chunks_ > 0x7fffffffull) throw std::invalid_argument("a list of up to 16 TB");
    bytes_ += e.bytes;
    in_place_ = in_place_ && e.in == e.out;
    outputs_ = outputs_ && e.out;
    all_.push_back(e);
  }
  for (size_t i = 0; i < all_.size(); i += PER_LAUNCH) {
    Piece piece;
    Table& t = piece.table;
    t = Table();
    t.count = (int)std::min<size_t>(PER_LAUNCH, all_.size() - i);
    for (int k = 0; k < t.count; ++k) {
      t.e[k] = all_[i + k];
      t.e[k].first -= all_[i].first;
    }
    t.chunks = (uint32_t)((i + t.count < all_.size() ? all_[i + t.count].first : chunks_) - all_[i].first);
    piece.at = partials_;
    partials_ += std::min<uint32_t>(t.chunks, MAX_BLOCKS);
    pieces_.push_back(piece);
  }
}

std::string ClipList::table() const {
  if (pieces_.size() < 2) return std::string();
  std::string s(reinterpret_cast<const char*>(all_.data()), all_.size() * sizeof(ClipEntry));
  std::vector<uint32_t> map(chunks_);
  for (size_t i = 0; i < all_.size(); ++i)
    std::fill(map.begin() + all_[i].first, i + 1 < all_.size() ? map.begin() + all_[i + 1].first : map.end(), (uint32_t)i);
  return s + std::string(reinterpret_cast<const char*>(map.data()), map.size() * sizeof(uint32_t));
}

namespace {

Resident resident_table(const void* at, size_t entries, uint64_t chunks) {
  Resident r;
  r.e = reinterpret_cast<const ClipEntry*>(at);
  r.map = reinterpret_cast<const uint32_t*>(r.e + entries);
  r.n = (uint32_t)chunks;
  return r;
}
int list_blocks(uint64_t chunks) { return (int)std::min<uint64_t>(chunks, MAX_BLOCKS); }

}  // namespace

void ClipList::norm(const void* resident, double* ws, hipStream_t s) const {
  // a list that the cache holds is read through it; of a larger one, the end is
  const uint32_t cold = bytes_ <= CACHE_BYTES ? 0 : (uint32_t)((bytes_ - CACHE_BYTES) / CHUNK_BYTES);
  if (resident) {
    hipLaunchKernelGGL(norm_kernel<Resident>, dim3(list_blocks(chunks_)), dim3(TPB), 0, s,
                       resident_table(resident, all_.size(), chunks_), cold, ws);
    return;
  }
  uint64_t before = 0;
  for (const Piece& p : pieces_) {
    const uint32_t c = cold > before ? (uint32_t)(cold - before) : 0;
    hipLaunchKernelGGL(norm_kernel<Inline>, dim3(list_blocks(p.table.chunks)), dim3(TPB), 0, s, Inline{p.table}, c,
                       ws + p.at);
    before += p.table.chunks;
  }
}

int ClipList::partials(const void* resident) const { return resident ? list_blocks(chunks_) : (int)partials_; }

void ClipList::finish(const void* resident, const double* ws, float* norm, hipStream_t s) const {
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(TPB), 0, s, ws, partials(resident), norm);
}

void ClipList::scale(const void* resident, double* ws, const float* use_norm, float clip, float* norm,
                     hipStream_t s) const {
  if (!(clip > 0.f)) throw std::invalid_argument("clip: the clip norm has to be positive");
  if (all_.empty()) {
    if (!use_norm) finish(resident, ws, norm, s);
    return;
  }
  if (!outputs_) throw std::invalid_argument("clip: a list without outputs");
  // results that would drive the rest of the list out of the cache go past it
  const int nt = 2 * bytes_ > CACHE_BYTES;
  int count = partials(resident);
  if (!use_norm && !resident && pieces_.size() > 1) {
    hipLaunchKernelGGL(fold_kernel, dim3(1), dim3(FOLD_TPB), 0, s, ws, count);
    count = 1;
  }
  if (resident) {
    hipLaunchKernelGGL(scale_kernel<Resident>, dim3(list_blocks(chunks_)), dim3(TPB), 0, s,
                       resident_table(resident, all_.size(), chunks_), ws, count, use_norm, clip, norm, (int)in_place_, nt);
    return;
  }
  for (size_t k = pieces_.size(); k-- > 0;) {
    const Piece& p = pieces_[k];
    hipLaunchKernelGGL(scale_kernel<Inline>, dim3(list_blocks(p.table.chunks)), dim3(TPB), 0, s, Inline{p.table}, ws,
                       count, use_norm, clip, k + 1 == pieces_.size() ? norm : (float*)nullptr, (int)in_place_, nt);
  }
}

int clipped_sgd_blocks(size_t n) {
  const size_t want = (n / 4 + TPB - 1) / TPB;
  return (int)std::min<size_t>(std::max<size_t>(want, 1), SGD_BLOCKS);
}

void launch_clipped_sgd_momentum_l2(float* p, const float* g, float* v, const float* l2x2, size_t n, float lr,
                                    float momentum, float grad_scale, float clip, const float* skip, double* ws,
                                    float* norm, hipStream_t s) {
  if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)v | (uintptr_t)l2x2) & 15)
    throw std::invalid_argument("clipped sgd: buffers must be 16-byte aligned");
  if (!(clip > 0.f)) throw std::invalid_argument("clipped sgd: the clip norm has to be positive");
  const int blocks = clipped_sgd_blocks(n);
  // three buffers are read for the norm: what of them the cache can keep for the update is read through it
  const size_t keep = CACHE_BYTES / 48, n4 = n / 4, cold = n4 > keep ? n4 - keep : 0;
  hipLaunchKernelGGL(sgd_norm_kernel, dim3(blocks), dim3(TPB), 0, s, p, g, l2x2, n, grad_scale, skip, cold, ws);
  hipLaunchKernelGGL(clipped_sgd_kernel, dim3(blocks), dim3(TPB), 0, s, p, g, v, l2x2, n, lr, momentum, grad_scale,
                     clip, skip, ws, blocks, norm, (int)(n4 * 96 > (size_t)CACHE_BYTES));
}
