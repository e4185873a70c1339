// Global gradient norm, clipping to it, and the momentum update with the clipped gradient.
//
//   norm = sqrt(sum over all tensors of g^2)      out = g * min(1, clip / norm)
//
// Two launches: the first leaves a partial sum per block, in the second every block adds the few hundred partial
// sums itself (in a fixed order, so a third launch, a ticket and atomics are not needed and the bits are the same
// every time) and scales.  Both are sweeps bound by memory; the second walks from the end, where the first has left
// the memory-side cache filled.
//
// Squares are taken and summed in 64 bits: they cannot overflow or vanish for any fp32 or bf16 gradient, and a sum
// of hundreds of millions keeps its digits; the sweeps are bound by memory all the same.
//
// A norm that is infinite or NaN makes every result NaN, as TensorFlow's clip_by_global_norm has it; a norm of zero
// leaves the gradients alone.
//
// Tensors come as a table in the kernel's arguments: nothing to upload and keep alive, and a captured launch holds
// its own copy.  The list is cut into chunks of 16 KB that never cross a tensor; a block takes a run of consecutive chunks.
#include <stdexcept>

#include "grad_clip.h"

namespace {

constexpr int TPB = 256;
constexpr int CHUNK_BYTES = TPB * 16 * 4;
constexpr int MAX_BLOCKS = 2048;      // per launch: eight blocks a CU, all its waves

struct __attribute__((packed, aligned(2))) Any16 { u32x4 v; };

template <int DT> struct Vec { static constexpr int N = DT == DT_F32 ? 4 : 8; };

template <int DT>
__device__ __forceinline__ void unpack(const u32x4 v, float* f) {
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
}
template <int DT>
__device__ __forceinline__ u32x4 pack(const float* f) {
  u32x4 v;
  if constexpr (DT == DT_F32) {
    v.x = __float_as_uint(f[0]); v.y = __float_as_uint(f[1]); v.z = __float_as_uint(f[2]); v.w = __float_as_uint(f[3]);
  } else {
    v.x = pack2<DT>(f[0], f[1]); v.y = pack2<DT>(f[2], f[3]); v.z = pack2<DT>(f[4], f[5]); v.w = pack2<DT>(f[6], f[7]);
  }
  return v;
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

// The tensor that chunk `c` lies in.
__device__ __forceinline__ int find(const ClipList::Table& t, uint32_t c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int DT>
__device__ __forceinline__ double chunk_squares(const void* in, int64_t n, uint32_t chunk) {
  typedef typename Elem<DT>::T T;
  constexpr int V = Vec<DT>::N;
  const int64_t at = (int64_t)chunk * (TPB * 4 * V) + (int64_t)threadIdx.x * V;
  const T* p = reinterpret_cast<const T*>(in);
  float f[4][V];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t e = at + (int64_t)k * TPB * V;
    if (e + V <= n) {
      unpack<DT>(reinterpret_cast<const Any16*>(p + e)->v, f[k]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[k][j] = e + j < n ? to_f<DT>(p[e + j]) : 0.f;
    }
  }
  double s[2] = {0., 0.};
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) s[j & 1] = fma((double)f[k][j], (double)f[k][j], s[j & 1]);
  return s[0] + s[1];
}

template <int DT>
__device__ __forceinline__ void chunk_scale(const void* in, void* out, int64_t n, uint32_t chunk, float factor) {
  typedef typename Elem<DT>::T T;
  constexpr int V = Vec<DT>::N;
  const int64_t at = (int64_t)chunk * (TPB * 4 * V) + (int64_t)threadIdx.x * V;
  const T* p = reinterpret_cast<const T*>(in);
  T* q = reinterpret_cast<T*>(out);
  u32x4 raw[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t e = at + (int64_t)k * TPB * V;
    if (e + V <= n) raw[k] = reinterpret_cast<const Any16*>(p + e)->v;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t e = at + (int64_t)k * TPB * V;
    if (e + V <= n) {
      float f[V];
      unpack<DT>(raw[k], f);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] *= factor;
      reinterpret_cast<Any16*>(q + e)->v = pack<DT>(f);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e + j < n) q[e + j] = from_f<DT>(to_f<DT>(p[e + j]) * factor);
    }
  }
}

constexpr int DT_SHIFT = 60;

__global__ __launch_bounds__(TPB) void norm_kernel(const ClipList::Table t, double* __restrict__ ws) {
  __shared__ double red[4];
  const uint32_t chunks = t.first[t.count];
  const uint32_t c0 = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x);
  const uint32_t c1 = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
  double s = 0.;
  int i = c0 < c1 ? find(t, c0) : 0;
  for (uint32_t c = c0; c < c1; ++c) {
    while (c >= t.first[i + 1]) ++i;
    const int64_t tag = t.n[i], n = tag & ((1ll << DT_SHIFT) - 1);
    const uint32_t k = c - t.first[i];
    switch ((int)(tag >> DT_SHIFT)) {
      case DT_BF16: s += chunk_squares<DT_BF16>(t.in[i], n, k); break;
      case DT_F16: s += chunk_squares<DT_F16>(t.in[i], n, k); break;
      default: s += chunk_squares<DT_F32>(t.in[i], n, k); break;
    }
  }
  s = block_sum64(s, red);
  if (threadIdx.x == 0) ws[blockIdx.x] = s;
}

__global__ __launch_bounds__(TPB) void norm_finish_kernel(const double* __restrict__ ws, int partials, float* norm) {
  __shared__ double red[4];
  (void)clip_factor(ws, partials, nullptr, 1.f, norm, red);
}

__global__ __launch_bounds__(TPB) void scale_kernel(const ClipList::Table t, const double* __restrict__ ws,
                                                    int partials, const float* __restrict__ use_norm, float clip,
                                                    float* norm, int in_place) {
  __shared__ double red[4];
  const float factor = clip_factor(ws, partials, use_norm, clip, norm, red);
  if (in_place && factor == 1.f) return;        // every result is where it belongs already
  const uint32_t chunks = t.first[t.count], b = gridDim.x - 1 - blockIdx.x;
  const uint32_t c0 = (uint32_t)((uint64_t)chunks * b / gridDim.x);
  const uint32_t c1 = (uint32_t)((uint64_t)chunks * (b + 1) / gridDim.x);
  int i = c0 < c1 ? find(t, c1 - 1) : 0;
  for (uint32_t c = c1; c-- > c0;) {
    while (c < t.first[i]) --i;
    const int64_t tag = t.n[i], n = tag & ((1ll << DT_SHIFT) - 1);
    const uint32_t k = c - t.first[i];
    switch ((int)(tag >> DT_SHIFT)) {
      case DT_BF16: chunk_scale<DT_BF16>(t.in[i], t.out[i], n, k, factor); break;
      case DT_F16: chunk_scale<DT_F16>(t.in[i], t.out[i], n, k, factor); break;
      default: chunk_scale<DT_F32>(t.in[i], t.out[i], n, k, factor); break;
    }
  }
}

// ---- the update ---------------------------------------------------------------------------------
//   g' = g * grad_scale + l2x2 * w      f = min(1, clip / |g'|)      v = momentum v - lr f g'      w += v
// (the norm is that of the whole gradient, the regulariser's part included, as an optimizer sees it)

__device__ __forceinline__ void unscale(const float* skip, float* grad_scale) {
  if (skip) *grad_scale *= skip[1];
}

__global__ __launch_bounds__(TPB) void sgd_norm_kernel(const float* __restrict__ p, const float* __restrict__ g,
                                                       const float* __restrict__ l2x2, size_t n, float grad_scale,
                                                       const float* __restrict__ skip, double* __restrict__ ws) {
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
  size_t i = blockIdx.x * (size_t)TPB + threadIdx.x;
  for (; i + 3 * stride < n4; i += 4 * stride) {       // twelve loads under way
    f32x4 w[4], gr[4], l2[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = reinterpret_cast<const f32x4*>(p)[i + k * stride];
      gr[k] = reinterpret_cast<const f32x4*>(g)[i + k * stride];
      l2[k] = reinterpret_cast<const f32x4*>(l2x2)[i + k * stride];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) take(w[k], gr[k], l2[k]);
  }
  for (; i < n4; i += stride)
    take(reinterpret_cast<const f32x4*>(p)[i], reinterpret_cast<const f32x4*>(g)[i], reinterpret_cast<const f32x4*>(l2x2)[i]);
  const size_t t = n4 * 4 + threadIdx.x;
  if (blockIdx.x == 0 && t < n) {
    const double d = (double)(g[t] * grad_scale + l2x2[t] * p[t]);
    s[0] = fma(d, d, s[0]);
  }
  const double sum = block_sum64((s[0] + s[1]) + (s[2] + s[3]), red);
  if (threadIdx.x == 0) ws[blockIdx.x] = sum;
}

__global__ __launch_bounds__(TPB) void clipped_sgd_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                          float* __restrict__ v, const float* __restrict__ l2x2,
                                                          size_t n, float lr, float momentum, float grad_scale,
                                                          float clip, const float* __restrict__ skip,
                                                          const double* __restrict__ ws, int partials, float* norm) {
  __shared__ double red[4];
  unscale(skip, &grad_scale);
  const float factor = clip_factor(ws, partials, nullptr, clip, norm, red);
  if (skip && skip[0] != 0.f) return;       // a gradient is not finite: the step is left out
  const float step = lr * factor;
  const size_t n4 = n / 4, stride = (size_t)gridDim.x * TPB;
  const size_t first = blockIdx.x * (size_t)TPB + threadIdx.x;
  if (blockIdx.x == 0 && n4 * 4 + threadIdx.x < n) {
    const size_t t = n4 * 4 + threadIdx.x;
    const float w = p[t], d = g[t] * grad_scale + l2x2[t] * w;
    float vel = -(d * step);
    if (momentum != 0.f) { vel = v[t] * momentum - d * step; v[t] = vel; }
    p[t] = w + vel;
  }
  for (size_t k = first; k < n4; k += stride) {
    const size_t i = n4 - 1 - k;
    f32x4 w = reinterpret_cast<const f32x4*>(p)[i];
    const f32x4 gr = reinterpret_cast<const f32x4*>(g)[i], l2 = reinterpret_cast<const f32x4*>(l2x2)[i];
    const f32x4 d = gr * grad_scale + l2 * w;
    if (momentum != 0.f) {
      f32x4 vel = reinterpret_cast<const f32x4*>(v)[i];
      vel = vel * momentum - d * step;
      reinterpret_cast<f32x4*>(v)[i] = vel;
      w += vel;
    } else {
      w -= d * step;
    }
    reinterpret_cast<f32x4*>(p)[i] = w;
  }
}

int elem_bytes(int dt) { return dt == DT_F32 ? 4 : 2; }

}  // namespace

ClipList::ClipList(const std::vector<ClipTensor>& tensors) {
  size_t i = 0;
  while (i < tensors.size()) {
    Piece piece;
    Table& t = piece.table;
    t = Table();
    uint64_t chunks = 0;
    for (; i < tensors.size() && t.count < PER_LAUNCH; ++i) {
      const ClipTensor& x = tensors[i];
      if (x.dt != DT_BF16 && x.dt != DT_F16 && x.dt != DT_F32) throw std::invalid_argument("unknown element type");
      if (x.n < 0 || x.n >= (1ll << 40)) throw std::invalid_argument("a tensor of up to 2^40 elements");
      if (x.n == 0) continue;
      const uint64_t mine = ((uint64_t)x.n * elem_bytes(x.dt) + CHUNK_BYTES - 1) / CHUNK_BYTES;
      if (chunks + mine > 0xfffffff0ull) {
        if (t.count == 0) throw std::invalid_argument("a tensor is too large");
        break;
      }
      t.in[t.count] = x.in;
      t.out[t.count] = x.out;
      t.n[t.count] = x.n | ((int64_t)x.dt << DT_SHIFT);
      t.first[t.count] = (uint32_t)chunks;
      chunks += mine;
      ++t.count;
    }
    if (t.count == 0) continue;
    t.first[t.count] = (uint32_t)chunks;
    piece.blocks = (int)(chunks < (uint64_t)MAX_BLOCKS ? chunks : (uint64_t)MAX_BLOCKS);
    piece.at = partials_;
    partials_ += piece.blocks;
    pieces_.push_back(piece);
  }
}

void ClipList::norm(double* ws, hipStream_t s) const {
  for (const Piece& p : pieces_)
    hipLaunchKernelGGL(norm_kernel, dim3(p.blocks), dim3(TPB), 0, s, p.table, ws + p.at);
}

void ClipList::finish(const double* ws, float* norm, hipStream_t s) const {
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(TPB), 0, s, ws, (int)partials_, norm);
}

void ClipList::scale(const double* ws, const float* use_norm, float clip, float* norm, hipStream_t s) const {
  if (pieces_.empty()) {
    if (!use_norm) finish(ws, norm, s);
    return;
  }
  for (size_t k = pieces_.size(); k-- > 0;) {
    const Piece& p = pieces_[k];
    bool in_place = true;
    for (int i = 0; i < p.table.count; ++i) {
      if (!p.table.out[i]) throw std::invalid_argument("clip: a list without outputs");
      in_place = in_place && p.table.out[i] == p.table.in[i];
    }
    hipLaunchKernelGGL(scale_kernel, dim3(p.blocks), dim3(TPB), 0, s, p.table, ws, (int)partials_, use_norm, clip,
                       k + 1 == pieces_.size() ? norm : (float*)nullptr, (int)in_place);
  }
}

int clipped_sgd_blocks(size_t n) {
  const size_t want = (n / 4 + TPB - 1) / TPB;
  return (int)(want < 1 ? 1 : want < 1024 ? want : 1024);
}

void launch_clipped_sgd_momentum_l2(float* p, const float* g, float* v, const float* l2x2, size_t n, float lr,
                                    float momentum, float grad_scale, float clip, const float* skip, double* ws,
                                    float* norm, hipStream_t s) {
  if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)v | (uintptr_t)l2x2) & 15)
    throw std::invalid_argument("clipped sgd: buffers must be 16-byte aligned");
  if (!(clip > 0.f)) throw std::invalid_argument("clipped sgd: the clip norm has to be positive");
  const int partials = clipped_sgd_blocks(n);
  hipLaunchKernelGGL(sgd_norm_kernel, dim3(partials), dim3(TPB), 0, s, p, g, l2x2, n, grad_scale, skip, ws);
  const size_t want = (n / 4 + TPB - 1) / TPB;
  const int blocks = (int)(want < 1 ? 1 : want < 2048 ? want : 2048);
  hipLaunchKernelGGL(clipped_sgd_kernel, dim3(blocks), dim3(TPB), 0, s, p, g, v, l2x2, n, lr, momentum, grad_scale,
                     clip, skip, ws, partials, norm);
}
