// The seam between two residual blocks, forward and backward.
//
//   n = N(y) * post_gamma + post_beta          (n = y without post_gamma)
//   h = x + scale * a(gate) * n                (a: identity or sigmoid; h = x without y)
//   z = N(h) * pre_gamma + pre_beta            (the next block's input; none without pre_gamma)
//
// N normalises a row over its C channels: v / sqrt(mean v^2 + eps), or with `layer` (v - mean) / sqrt(var + eps).
// Rows are pixels of an NHWC activation or tokens.  The work is a handful of operations per element, so memory
// bounds it: every tensor is read once and written once, a row stays in registers (fp32) between its two
// normalisations, and nothing but results goes back to memory.  z is taken from the unrounded h.
//
// Split: a lane owns eight consecutive channels (16 bytes of a 16-bit row).  Rows of up to 512 channels share a
// wave (2 .. 64 lanes a row, sums by butterfly); wider rows take as many waves as they need, up to eight with one
// or two chunks of eight channels a lane, and join their sums through LDS.
//
// Loads and stores take any alignment (rows of odd length start anywhere).
//
// Measured, calls one behind the other: 200704 x 512 bf16 forward with a gate per image 148 us (5.6 TB/s), gradient with a
// sigmoid gate per element 281 us (5.9 TB/s; a copy of 1 GB 5.0); 12544 x 2048 bf16 forward, layer, scale per channel 40 us,
// gradient with a gate per image 67 us, of which its two kernels take 61 and 5; one row of 4096 9.8 us, its kernel 3.3.
//
// A file per element type instantiates these (residual_norm_bf16 / f16 / f32.hip).
#pragma once
#include <algorithm>
#include <stdexcept>

#include "residual_norm.h"

namespace rn {

// 16 bytes at the alignment of their elements: the memory system takes any address, one load all the same
typedef u32x4 __attribute__((aligned(2))) Any16;
typedef f32x4 __attribute__((aligned(4))) Any16F;

// NT: past the caches (a sweep over more than they hold)
template <bool NT, typename V>
__device__ __forceinline__ V get16(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool NT, typename V, typename W>
__device__ __forceinline__ void put16(V* p, const W v) {
  if constexpr (NT) __builtin_nontemporal_store((V)v, p);
  else *p = v;
}

// Moves the eight elements down by `n` (1 .. 7); zeros follow.
template <int DT>
__device__ __forceinline__ void move_down(Raw8<DT>& r, int n) {
  if constexpr (DT == DT_F32) {
    float f[8] = {r.lo[0], r.lo[1], r.lo[2], r.lo[3], r.hi[0], r.hi[1], r.hi[2], r.hi[3]};
#pragma unroll
    for (int by = 4; by; by >>= 1)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = !(n & by) ? f[j] : j + by < 8 ? f[j + by] : 0.f;
    r.lo = f32x4{f[0], f[1], f[2], f[3]};
    r.hi = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    uint32_t w[5] = {r.v.x, r.v.y, r.v.z, r.v.w, 0u};
#pragma unroll
    for (int by = 2; by; by >>= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = !((n >> 1) & by) ? w[j] : j + by < 4 ? w[j + by] : 0u;
    if (n & 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (w[j] >> 16) | (w[j + 1] << 16);
    }
    r.v = u32x4{w[0], w[1], w[2], w[3]};
  }
}

// Where a lane's eight channels from `c` on are loaded from.  The lane with a row's last, partial chunk reads the row's
// last eight elements in the same load as everyone else and moves them into place when they are used (`settle`); element
// by element its loads would be up to eight more trips to memory, one after the other.  Rows of fewer than eight
// channels (TINY kernels) have no such eight.
struct Chunk {
  int c, at;
};
__device__ __forceinline__ Chunk chunk_of(int c, int C) { return Chunk{c, C < 8 ? c : min(c, C - 8)}; }

// The chunk as it sits in memory (a partial one still to be settled), zeros in lanes past the row's end and where the
// row is not there (`live`).
template <int DT, bool NT, bool TINY>
__device__ __forceinline__ Raw8<DT> load_raw(const typename Elem<DT>::T* p, const Chunk& k, bool live, int C) {
  Raw8<DT> r = zero_raw<DT>();
  if (live && k.c < C) {
    if (!TINY || C >= 8) {
      if constexpr (DT == DT_F32) {
        r.lo = get16<NT>(reinterpret_cast<const Any16F*>(p + k.at));
        r.hi = get16<NT>(reinterpret_cast<const Any16F*>(p + k.at + 4));
      } else {
        r.v = get16<NT>(reinterpret_cast<const Any16*>(p + k.at));
      }
    } else if constexpr (DT == DT_F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (k.c + j < C) r.lo[j] = p[k.c + j];
        if (k.c + 4 + j < C) r.hi[j] = p[k.c + 4 + j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k.c + j < C) r.v[j >> 1] |= (uint32_t)p[k.c + j] << (16 * (j & 1));
    }
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void settle(Raw8<DT>& r, const Chunk& k, int C) {
  if (k.c < C && k.at != k.c) move_down<DT>(r, k.c - k.at);
}

// MODE of a row kernel.  The common calls - every tensor there, rows of whole chunks, one chunk a lane - get kernels
// whose loads are all unconditional (FULL): only then does the compiler know how many loads are under way, and waiting for a
// row does not wait for the one asked for after it.  Everything else goes through kernels that look what is there
// (any tensor may be missing, any row length).
enum Mode { ANY = 0, ANY_GROUP = 1, FULL_PLAIN = 2, FULL_GROUP = 3, FULL_ELEMENT = 4 };

// FULL: the lane's chunk, of some row that is there; lanes past the row's end read its last chunk again (`drop`ped later).
template <int DT, bool NT>
__device__ __forceinline__ Raw8<DT> full_raw(const void* p, int64_t at) {
  Raw8<DT> r;
  if constexpr (DT == DT_F32) {
    const Any16F* q = reinterpret_cast<const Any16F*>(reinterpret_cast<const float*>(p) + at);
    r.lo = get16<NT>(q);
    r.hi = get16<NT>(q + 1);
  } else {
    r.v = get16<NT>(reinterpret_cast<const Any16*>(reinterpret_cast<const uint16_t*>(p) + at));
  }
  return r;
}
template <int DT>
__device__ __forceinline__ void drop(Raw8<DT>& r, bool keep) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { r.lo[j] = keep ? r.lo[j] : 0.f; r.hi[j] = keep ? r.hi[j] : 0.f; }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = keep ? r.v[j] : 0u;
  }
}

template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* p, int c, int C, float* f) {
  const Chunk k = chunk_of(c, C);
  Raw8<DT> r = load_raw<DT, false, true>(p, k, true, C);
  settle<DT>(r, k, C);
  unpack8<DT>(r, f);
}

template <int DT, bool NT = false, bool ODD = true>
__device__ __forceinline__ void store8(typename Elem<DT>::T* p, int c, int C, const float* f) {
  if (c + 8 <= C) {
    if constexpr (DT == DT_F32) {
      put16<NT>(reinterpret_cast<Any16F*>(p + c), f32x4{f[0], f[1], f[2], f[3]});
      put16<NT>(reinterpret_cast<Any16F*>(p + c + 4), f32x4{f[4], f[5], f[6], f[7]});
    } else {
      u32x4 v;
      v.x = pack2<DT>(f[0], f[1]); v.y = pack2<DT>(f[2], f[3]);
      v.z = pack2<DT>(f[4], f[5]); v.w = pack2<DT>(f[6], f[7]);
      put16<NT>(reinterpret_cast<Any16*>(p + c), v);
    }
  } else if constexpr (ODD) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < C) p[c + j] = from_f<DT>(f[j]);
  }
}

// Rows of the results.
template <int DT, bool NT, bool ODD>
__device__ __forceinline__ void store_row(void* to, int64_t at, int c, int C, const float* f) {
  typename Elem<DT>::T* p = reinterpret_cast<typename Elem<DT>::T*>(to) + at;
  store8<DT, NT, ODD>(p, c, C, f);
}

// A sigmoid gate's factor and its derivative, the latter as e / (1 + e)^2 with e = exp(-|g|): a (1 - a) of a rounded a
// has lost its digits from g = 8 on (6 % at 16, everything at 18).
//
// EXACT: the library's exponential and a true division.  The hardware's are off by up to (|g| + 8) 2^-24 of their value.
// They serve where a 16-bit value per element is gated and the result is rounded to 16 bits again: the forward pass, and
// in the gradient of a gate per element dy and dgate; the terms of that call's sums over rows carry the same error
// into dpost_gamma and dpost_beta, next to the 2^-11 or 2^-8 that their 16-bit factors have been rounded by.  A gate of groups
// is fp32 whatever the rows are: its gradient is computed EXACT.
struct Sigmoid {
  float a, slope;
};
template <bool EXACT>
__device__ __forceinline__ Sigmoid sigmoid_f(float g) {
  const float e = EXACT ? expf(-fabsf(g)) : __expf(-fabsf(g));
  const float d = EXACT ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e);
  return Sigmoid{g < 0.f ? e * d : d, e * d * d};
}

// v + v of the lane that is `O` away, in every lane (O = 1, 2, 4 .. 32 in this order: from O = 4 on the lanes of the
// smaller groups hold the same value already, so a mirrored row does for an exchange).  Register to register: no trip
// through LDS.
template <int O>
__device__ __forceinline__ float add_lane(float v) {
  const int i = __float_as_int(v);
  if constexpr (O == 1) return v + __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0xB1, 0xf, 0xf, true));
  else if constexpr (O == 2) return v + __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0x4E, 0xf, 0xf, true));
  else if constexpr (O == 4) return v + __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0x141, 0xf, 0xf, true));
  else if constexpr (O == 8) return v + __int_as_float(__builtin_amdgcn_update_dpp(0, i, 0x140, 0xf, 0xf, true));
  else if constexpr (O == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(i, i, false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(i, i, false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
  }
}

// What the waves of a wide row leave for each other: [turn][value][wave], zero where there is no wave.
typedef float Red[2][4][8];

template <bool WIDE>
__device__ __forceinline__ void clear_red(Red red) {
  if constexpr (WIDE) {
    if (threadIdx.x < 64) (&red[0][0][0])[threadIdx.x] = 0.f;
    __syncthreads();
  }
}

// Sums of N values over the lanes of a row, given to all of them.  LPR lanes of a wave hold a narrow row; a wide one
// has up to eight waves, joined through the half `turn & 1` of `red`: the barrier of the next sum separates this
// sum's reads from the writes after next.  Every eight lanes read the eight waves' values and add them among
// themselves: one trip to LDS for all values (a loop over the waves makes as many trips as there are waves).
template <int LPR, bool WIDE, int N>
__device__ __forceinline__ void row_sums(float* v, Red red, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = add_lane<1>(v[i]);
    if constexpr (LPR >= 4) v[i] = add_lane<2>(v[i]);
    if constexpr (LPR >= 8) v[i] = add_lane<4>(v[i]);
    if constexpr (LPR >= 16) v[i] = add_lane<8>(v[i]);
    if constexpr (LPR >= 32) v[i] = add_lane<16>(v[i]);
    if constexpr (LPR >= 64) v[i] = add_lane<32>(v[i]);
  }
  if constexpr (WIDE) {
    float (*mine)[8] = red[turn & 1];
    ++turn;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine[i][threadIdx.x >> 6] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = mine[i][threadIdx.x & 7];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = add_lane<4>(add_lane<2>(add_lane<1>(v[i])));
  }
}

// Subtracts the mean of the row from its channels (and leaves those past the end zero).
template <int K, bool ODD>
__device__ __forceinline__ void centre(float (*v)[8], const int* c, int C, float mean) {
  if constexpr (!ODD) {       // a lane's channels are all there or none is
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float m = c[k] < C ? mean : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] -= m;
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = c[k] + j < C ? v[k][j] - mean : 0.f;
  }
}

// Centres `v` (LAYER) and returns 1 / sqrt(mean square + eps) of the row.
template <int LPR, bool WIDE, int K, bool LAYER, bool ODD>
__device__ __forceinline__ float normalise(float (*v)[8], const int* c, int C, float inv_c, float eps,
                                           Red red, int& turn) {
  float s[1];
  if constexpr (LAYER) {
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[0] += v[k][j];
    row_sums<LPR, WIDE, 1>(s, red, turn);
    centre<K, ODD>(v, c, C, s[0] * inv_c);
  }
  s[0] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) s[0] += v[k][j] * v[k][j];
  row_sums<LPR, WIDE, 1>(s, red, turn);
  return 1.f / sqrtf(s[0] * inv_c + eps);
}

template <int DT, int K>
struct FwdIn {
  Raw8<DT> x[K], y[K], gate[K];
  Raw8<DT_F32> group[K];
};

template <int DT, int K, bool NT, bool TINY>
__device__ __forceinline__ void load_fwd(FwdIn<DT, K>& in, const ResidualNormParams& p, int64_t r, bool live,
                                         const Chunk* at) {
  typedef typename Elem<DT>::T T;
  const int C = p.C;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.x[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.x) + r * p.ldx, at[k], live, C);
    if (p.y) in.y[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.y) + r * p.ldy, at[k], live, C);
    if (p.gate_mode == GATE_ELEMENT)
      in.gate[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.gate) + r * p.ldgate, at[k], live, C);
    if (p.gate_mode == GATE_GROUP)
      in.group[k] = load_raw<DT_F32, false, TINY>(reinterpret_cast<const float*>(p.gate) +
                                                      (int64_t)((uint32_t)r / (uint32_t)p.group_rows) * p.ldgate,
                                                  at[k], live, C);
  }
}

template <int DT, int K>
__device__ __forceinline__ void settle_row(FwdIn<DT, K>& in, const ResidualNormParams& p, const Chunk* at) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    settle<DT>(in.x[k], at[k], p.C);
    if (p.y) settle<DT>(in.y[k], at[k], p.C);
    if (p.gate_mode == GATE_ELEMENT) settle<DT>(in.gate[k], at[k], p.C);
    if (p.gate_mode == GATE_GROUP) settle<DT_F32>(in.group[k], at[k], p.C);
  }
}

template <int DT, int K, bool NT, int MODE>
__device__ __forceinline__ void load_full(FwdIn<DT, K>& in, const ResidualNormParams& p, int64_t r, const Chunk* at) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.x[k] = full_raw<DT, NT>(p.x, r * p.ldx + at[k].at);
    in.y[k] = full_raw<DT, NT>(p.y, r * p.ldy + at[k].at);
    if constexpr (MODE == FULL_ELEMENT) in.gate[k] = full_raw<DT, NT>(p.gate, r * p.ldgate + at[k].at);
    if constexpr (MODE == FULL_GROUP)
      in.group[k] = full_raw<DT_F32, false>(p.gate, (int64_t)((uint32_t)r / (uint32_t)p.group_rows) * p.ldgate + at[k].at);
  }
}

// The blocks walk the rows side by side: while one row's sums are taken the next one's loads are under way, and the
// vectors stay in registers.
// Waves per SIMD that the registers are kept small enough for.
constexpr int fwd_waves(int dt, bool layer, int chunks) { return chunks > 1 ? 2 : layer && dt == DT_F32 ? 3 : 4; }

template <int DT, int LPR, bool WIDE, int K, bool LAYER, int MODE, bool NT>
__global__ __launch_bounds__(WIDE ? 512 : 256, fwd_waves(DT, LAYER, K)) void fwd_kernel(const ResidualNormParams p) {
  constexpr bool FULL = MODE >= FULL_PLAIN, ODD = !FULL;
  __shared__ Red red;
  clear_red<WIDE>(red);
  int turn = 0;
  const int lanes = WIDE ? (int)blockDim.x : LPR;
  const int lane = WIDE ? (int)threadIdx.x : (int)(threadIdx.x % LPR);
  const int slots = WIDE ? 1 : 256 / LPR;
  const int slot = WIDE ? 0 : (int)(threadIdx.x / LPR);
  const int C = p.C;
  const float inv_c = 1.f / (float)C;
  int c[K];
  Chunk at[K];
  float pw[K][8], pb[K][8], qw[K][8], qb[K][8], g[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    c[k] = (lane + k * lanes) * 8;
    at[k] = chunk_of(c[k], C);
#pragma unroll
    for (int j = 0; j < 8; ++j) { pw[k][j] = pb[k][j] = qw[k][j] = qb[k][j] = 0.f; g[k][j] = 1.f; }
    if (p.post_gamma) load8<DT_F32>(p.post_gamma, c[k], C, pw[k]);
    if (LAYER && p.post_beta) load8<DT_F32>(p.post_beta, c[k], C, pb[k]);
    if (p.pre_gamma) load8<DT_F32>(p.pre_gamma, c[k], C, qw[k]);
    if (LAYER && p.pre_beta) load8<DT_F32>(p.pre_beta, c[k], C, qb[k]);
  }
  // every lane of a wave walks the same number of passes (the sums need all of them); a row past the run's end has
  // no channels: zeros are read and nothing is written for it
  const int64_t row0 = (int64_t)blockIdx.x * slots, row1 = p.P, step = (int64_t)gridDim.x * slots;
  const bool has_y = FULL || p.y;
  const int gate_mode = MODE == FULL_PLAIN ? (int)GATE_NONE : MODE == FULL_GROUP ? (int)GATE_GROUP :
                        MODE == FULL_ELEMENT ? (int)GATE_ELEMENT : p.gate_mode;
  auto work = [&](FwdIn<DT, K>& in, int64_t base) __attribute__((always_inline)) {
    const int64_t r = WIDE || base + slot < row1 ? base + slot : 0;
    const int Cr = WIDE || base + slot < row1 ? C : 0;
    float h[K][8], v[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) unpack8<DT>(in.x[k], h[k]);
    if (has_y) {
      if (gate_mode != GATE_NONE) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (gate_mode == GATE_GROUP) unpack8<DT_F32>(in.group[k], g[k]);
          else unpack8<DT>(in.gate[k], g[k]);
          if (p.sigmoid) {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[k][j] = sigmoid_f<DT == DT_F32>(g[k][j]).a;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) unpack8<DT>(in.y[k], v[k]);
      if (p.post_gamma) {
        const float rs = normalise<LPR, WIDE, K, LAYER, ODD>(v, c, Cr, inv_c, p.eps, red, turn);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = LAYER ? v[k][j] * rs * pw[k][j] + pb[k][j] : v[k][j] * rs * pw[k][j];
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[k][j] += p.scale * (g[k][j] * v[k][j]);
        store_row<DT, NT, ODD>(p.h, r * C, c[k], Cr, h[k]);
      }
    }
    if (p.pre_gamma) {
      const float rs = normalise<LPR, WIDE, K, LAYER, ODD>(h, c, Cr, inv_c, p.eps, red, turn);
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[k][j] = LAYER ? h[k][j] * rs * qw[k][j] + qb[k][j] : h[k][j] * rs * qw[k][j];
        store_row<DT, NT, ODD>(p.z, r * C, c[k], Cr, h[k]);
      }
    }
  };
  if constexpr (FULL) {
    // lanes past the row's end, slots past the last row
    const bool ragged = C != lanes * 8 || (!WIDE && p.P % slots != 0);
    auto ask = [&](int64_t base, FwdIn<DT, K>& to) __attribute__((always_inline)) {
      const int64_t r = base + slot < row1 ? base + slot : 0;
      load_full<DT, K, NT, MODE>(to, p, r, at);
    };
    auto take = [&](FwdIn<DT, K>& in, int64_t base) __attribute__((always_inline)) {
      if (ragged) {
        const bool keep = c[0] < C && (WIDE || base + slot < row1);
        drop<DT>(in.x[0], keep);
        drop<DT>(in.y[0], keep);
        if constexpr (MODE == FULL_ELEMENT) drop<DT>(in.gate[0], keep);
        if constexpr (MODE == FULL_GROUP) drop<DT_F32>(in.group[0], keep);
      }
      work(in, base);
    };
    FwdIn<DT, K> a, b;       // two rows under way, in registers of their own: copying one would wait for it
    ask(row0, a);
    for (int64_t base = row0; base < row1; base += 2 * step) {
      ask(base + step, b);
      take(a, base);
      if (base + step >= row1) break;
      ask(base + 2 * step, a);
      take(b, base + step);
    }
  } else {
    FwdIn<DT, K> next;
    auto ask = [&](int64_t base) {
      if (base >= row1) return;
      const bool live = WIDE || base + slot < row1;
      const int64_t r = live ? base + slot : 0;
      load_fwd<DT, K, NT, LPR == 2>(next, p, r, live, at);
    };
    ask(row0);
    for (int64_t base = row0; base < row1; base += step) {
      FwdIn<DT, K> in = next;
      ask(base + step);                    // before anything waits for this row
      settle_row(in, p, at);
      work(in, base);
    }
  }
}

// ---- backward ----------------------------------------------------------------------------------
//   H  = dh + r_h (dz' - [mean dz'] - hat_h mean(dz' hat_h))        dz' = dz * pre_gamma,  hat_h = N(h)
//   dx = H        up = scale * H        dgate = up * n * a'(gate)   dn = up * a(gate)
//   dy = r_y (t - [mean t] - hat_y mean(t hat_y))                   t = dn * post_gamma,   hat_y = N(y)
//   dpre_gamma = sum dz hat_h   dpre_beta = sum dz   dpost_gamma = sum dn hat_y   dpost_beta = sum dn
// (the bracketed means only with `layer`).  The statistics are taken again from h and y, which are in registers
// anyway: two sums more per row instead of saved tensors that could belong to another call.
// A lane keeps its channels for all of its block's rows, so the sums over rows are registers; blocks leave one row of
// partial sums each and finish_kernel adds them in a fixed order (no atomics: the same bits every time).  A slot's sum over
// its rows is fp32 and so is a block's partial sum in memory; both joins add in 64 bits (131072 x 16 fp32 layer: 8.1e-8 off, as
// 64-bit sums over fp32 terms are, 1.9e-7 with fp32 joins; 1 % of the time of small calls).
//
// A block's rows lie in one group (of rows that share a gate row), or it owns whole groups; many groups of few rows each go
// to the row slots, each of which owns whole groups (`own_groups`).

struct BwdPlan {
  int blocks;        // grid
  int parts;         // blocks per group
  int groups;        // groups of rows (1 without a group gate)
  int group_rows;
  int own_groups;    // each row slot takes whole groups
  int nt;            // more bytes than the memory-side cache holds: loads and stores past the caches
};

// Waves per SIMD that the backward kernel is built for: its registers (sums over rows, vectors, a row in work and the
// next ones' loads) leave room for two, three for RMS norms of 16-bit rows.  (A FULL kernel with the sums of a group's
// gate besides would spill 6 - 12 registers at three, and its grids ask for two at most.)
constexpr int bwd_waves(int dt, bool layer, int chunks, int mode) {
  return !layer && dt != DT_F32 && chunks == 1 && mode != FULL_GROUP ? 3 : 2;
}

inline int narrow_lanes(int C) {       // lanes a row of up to 512 channels
  int l = 2;
  while (l * 8 < C) l *= 2;
  return l;
}

inline int wide_threads(int C) {
  const int per_wave = C <= 4096 ? 512 : 1024;
  return 64 * ((C + per_wave - 1) / per_wave);
}

// Whether `tensors` tensors of the rows are more than the 256 MB that the memory-side cache holds.
inline int big(const ResidualNormParams& p, int tensors) {
  return (int64_t)p.P * p.C * (p.dt == DT_F32 ? 4 : 2) * tensors > (256ll << 20);
}

// FULL kernels need every tensor, whole chunks and one chunk a lane.
inline bool full_rows(const ResidualNormParams& p) { return p.C % 8 == 0 && p.C <= 4096 && p.y; }

// How many waves a CU works on a sweep.  Over more than the cache holds a narrow front is best: eight (200704 x 512 bf16
// with a gate per image: 146 us, 156 with sixteen; 50000 x 2048 with a gate per element: 177 and 189), sixteen where
// no gate is read (100000 x 1024 bf16, layer: 152, 162 with eight).  What the cache holds wants sixteen (12544 x 2048 bf16,
// layer: 36 us, 45 with four; 6000 x 1024: 12.6, 24 with two), and a block for every row where there are few.
inline int fwd_blocks(const ResidualNormParams& p, int nt) {
  const int slots = p.C <= 512 ? 256 / narrow_lanes(p.C) : 1;
  const int waves = (p.C <= 512 ? 256 : wide_threads(p.C)) / 64;
  const int64_t want = ((int64_t)p.P + slots - 1) / slots;
  const int64_t most = 256 * std::max(1, (nt && p.gate_mode != GATE_NONE ? 8 : 16) / waves);
  return (int)(want <= (nt ? 1 : 4) * most ? want : most);
}

// `full`: the sweep runs on a FULL kernel.
inline BwdPlan plan_bwd(const ResidualNormParams& p, bool full) {
  BwdPlan b;
  const bool grouped = p.gate_mode == GATE_GROUP;
  b.group_rows = grouped ? p.group_rows : p.P;
  b.groups = p.P / b.group_rows;
  const int slots = p.C <= 512 ? 256 / narrow_lanes(p.C) : 1;
  const int waves = (p.C <= 512 ? 256 : wide_threads(p.C)) / 64;
  b.nt = big(p, 6);
  // Waves a CU: eight (6000 x 1024 bf16: 25 us, 41 with two; 3000 x 2048 layer: 27.5, 35 with twelve).  FULL kernels, with
  // two rows under way, run large sweeps best as a front of four (200704 x 512 with a gate per element: 277 us, 306 with
  // eight, before its sigmoid kept its digits; the last ResNet stage with a gate per image: 66 and 69, and a group's gate gradient stays in one block); the
  // others want all that are resident where their groups are many (12544 x 2047: 81 us, 90 with eight).
  const int resident = 4 * bwd_waves(p.dt, p.layer, p.C <= 4096 ? 1 : 2, ANY_GROUP);
  const int want = 256 * std::max(1, (b.nt && full ? 4 : b.nt && grouped ? resident : 8) / waves);
  // A slot that walks a group by itself takes 0.7 us a row however idle the rest is; a block that shares a group's rows
  // among its slots pays for joining them, about four rows' time a group.  bf16, 16 channels: 500 rows in one group 364 us a slot
  // for itself and 8.6 us shared, 4 x 256 10.4 and 10.9, 16 x 2000 20 and 26, 32 x 2000 33 and 26, 16 x 16000 25 and 78.
  // Long groups of their own also read far apart: 100 x 16000 303 and 166.
  const int sets = (b.groups + slots - 1) / slots;
  const int64_t alone = (int64_t)b.group_rows * ((sets + want - 1) / want);
  b.own_groups = grouped && slots > 1 && b.group_rows < 4 * slots && b.group_rows <= 32 &&
                 alone <= 4 * (int64_t)((b.groups + want - 1) / want);
  if (b.own_groups) {
    b.blocks = sets < want ? sets : want;
    b.parts = 1;
    return b;
  }
  b.parts = 1;
  if (b.groups == 1) {
    b.parts = std::min((b.group_rows + slots - 1) / slots, want);      // a part has work for every slot
    b.blocks = b.parts;
  } else if (b.groups < 4 * want) {
    // the parts that leave the busiest place on the grid the least work: rows, and about two rows' traffic for the
    // partial sums that a block leaves
    const int most = std::min((b.group_rows + slots - 1) / slots, 4 * want / b.groups);
    int64_t best = INT64_MAX;
    for (int parts = 1; parts <= std::max(1, most); ++parts) {
      const int64_t rounds = ((int64_t)b.groups * parts + want - 1) / want;
      const int64_t rows = (b.group_rows + (int64_t)parts * slots - 1) / ((int64_t)parts * slots);
      if (rounds * (rows + 2) < best) { best = rounds * (rows + 2); b.parts = parts; }
    }
    b.blocks = b.groups * b.parts;
  } else {
    b.blocks = want;
  }
  return b;
}

// Partial sums: [vector][block][C]; which vectors are kept goes by the gradients asked for.
struct Partials {
  float* row[5];      // dpre_gamma, dpost_gamma, dpre_beta, dpost_beta, dgate
};

// The tensors of a row as they sit in memory.
template <int DT, int K>
struct RowIn {
  Raw8<DT> dh[K], dz[K], h[K], y[K], gate[K];
};

template <int DT, int K, bool NT, bool TINY>
__device__ __forceinline__ void load_row(RowIn<DT, K>& in, const ResidualNormParams& p, int64_t r, bool live,
                                         const Chunk* at) {
  typedef typename Elem<DT>::T T;
  const int C = p.C;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.dh[k] = zero_raw<DT>();
    if (p.dh) in.dh[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.dh) + r * p.lddh, at[k], live, C);
    if (p.dz) {
      in.dz[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.dz) + r * p.lddz, at[k], live, C);
      in.h[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.x) + r * p.ldx, at[k], live, C);
    }
    if (p.y) in.y[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.y) + r * p.ldy, at[k], live, C);
    if (p.gate_mode == GATE_ELEMENT)
      in.gate[k] = load_raw<DT, NT, TINY>(reinterpret_cast<const T*>(p.gate) + r * p.ldgate, at[k], live, C);
  }
}

template <int DT, int K>
__device__ __forceinline__ void settle_row(RowIn<DT, K>& in, const ResidualNormParams& p, const Chunk* at) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (p.dh) settle<DT>(in.dh[k], at[k], p.C);
    if (p.dz) {
      settle<DT>(in.dz[k], at[k], p.C);
      settle<DT>(in.h[k], at[k], p.C);
    }
    if (p.y) settle<DT>(in.y[k], at[k], p.C);
    if (p.gate_mode == GATE_ELEMENT) settle<DT>(in.gate[k], at[k], p.C);
  }
}

template <int DT, int K, bool NT, int MODE>
__device__ __forceinline__ void load_full(RowIn<DT, K>& in, const ResidualNormParams& p, int64_t r, const Chunk* at) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    in.h[k] = full_raw<DT, NT>(p.x, r * p.ldx + at[k].at);
    in.dz[k] = full_raw<DT, NT>(p.dz, r * p.lddz + at[k].at);
    in.y[k] = full_raw<DT, NT>(p.y, r * p.ldy + at[k].at);
    in.dh[k] = full_raw<DT, NT>(p.dh, r * p.lddh + at[k].at);
    if constexpr (MODE == FULL_ELEMENT) in.gate[k] = full_raw<DT, NT>(p.gate, r * p.ldgate + at[k].at);
  }
}

// Sums the slots' eight channels a lane and hands every column's sum to `use(column, sum)`.  A thread adds eight slots,
// then the eighths are added (one thread a column and all 128 slots in turn took 1 us a vector for 16 channels).  In
// 64 bits: `sum` is rounded where it is stored, and `join` holds the eighths as doubles.
template <int LPR, typename F>
__device__ __forceinline__ void over_slots(const float* v, float* join, F use) {
  constexpr int COLS = LPR * 8, PARTS = COLS >= 256 ? 1 : 256 / COLS, SLOTS = 256 / LPR;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) join[(int)threadIdx.x * 8 + j] = v[j];
  __syncthreads();
  if constexpr (PARTS == 1) {
#pragma unroll
    for (int col = threadIdx.x; col < COLS; col += 256) {
      double sum = 0.;
#pragma unroll
      for (int q = 0; q < SLOTS; ++q) sum += join[q * COLS + col];
      use(col, sum);
    }
  } else {
    const int col = threadIdx.x % COLS, part = threadIdx.x / COLS;
    double sum = 0.;
#pragma unroll
    for (int q = 0; q < SLOTS / PARTS; ++q) sum += join[(part * (SLOTS / PARTS) + q) * COLS + col];
    __syncthreads();
    double* parts = reinterpret_cast<double*>(join);
    parts[threadIdx.x] = sum;
    __syncthreads();
    if (part == 0) {
      sum = 0.;
#pragma unroll
      for (int q = 0; q < PARTS; ++q) sum += parts[q * COLS + col];
      use(col, sum);
    }
  }
}

template <int DT, int LPR, bool WIDE, int K, bool LAYER, int MODE, bool NT>
__global__ __launch_bounds__(WIDE ? 512 : 256, bwd_waves(DT, LAYER, K, MODE)) void bwd_kernel(const ResidualNormParams p, const BwdPlan plan,
                                                               const Partials part) {
  typedef typename Elem<DT>::T T;
  constexpr bool FULL = MODE >= FULL_PLAIN, GROUP = MODE == ANY_GROUP || MODE == FULL_GROUP, ODD = !FULL;
  const bool has_dz = FULL || p.dz, has_y = FULL || p.y;
  const bool element = FULL ? MODE == FULL_ELEMENT : p.gate_mode == GATE_ELEMENT;
  // sums over rows: of the two gammas, with LAYER of the two betas, with GROUP of the gate
  constexpr int SUMS = 2 + (LAYER ? 2 : 0) + (GROUP ? 1 : 0), GATE = SUMS - 1;
  __shared__ Red red;
  clear_red<WIDE>(red);
  __shared__ __attribute__((aligned(8))) float join[WIDE ? 2 : 256 * 8];
  int turn = 0;
  const int lanes = WIDE ? (int)blockDim.x : LPR;
  const int lane = WIDE ? (int)threadIdx.x : (int)(threadIdx.x % LPR);
  const int slots = WIDE ? 1 : 256 / LPR;
  const int slot = WIDE ? 0 : (int)(threadIdx.x / LPR);
  const int C = p.C;
  const float inv_c = 1.f / (float)C;
  int c[K];
  Chunk at[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    c[k] = (lane + k * lanes) * 8;
    at[k] = chunk_of(c[k], C);
  }
  float acc[SUMS][K][8];
#pragma unroll
  for (int i = 0; i < SUMS; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][k][j] = 0.f;
  // post_gamma, post_beta, pre_gamma of the lane's channels: kept, or with two chunks a lane, whose sums alone take half
  // of the registers, read again for every row
  constexpr bool KEPT = K == 1;
  float pw[K][8], pb[K][8], qw[K][8];
  auto get_pre = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) qw[k][j] = 0.f;
      if (p.pre_gamma) load8<DT_F32>(p.pre_gamma, c[k], C, qw[k]);
    }
  };
  auto get_post = [&]() {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) { pw[k][j] = 1.f; pb[k][j] = 0.f; }
      if (p.post_gamma) load8<DT_F32>(p.post_gamma, c[k], C, pw[k]);
      if (LAYER && p.post_beta) load8<DT_F32>(p.post_beta, c[k], C, pb[k]);
    }
  };
  if (KEPT) { get_pre(); get_post(); }
  // the sets of groups this block works on, and the rows of a group that are its own
  const int per_set = plan.own_groups ? slots : 1;
  const int first_set = plan.parts > 1 ? (int)blockIdx.x / plan.parts : (int)blockIdx.x;
  const int stride_set = plan.parts > 1 ? plan.groups : (int)gridDim.x;      // parts > 1: one group a block
  const int sets = (plan.groups + per_set - 1) / per_set;
  const int row0 = plan.parts > 1 ? ((int)blockIdx.x % plan.parts) * slots : 0;
  const int row1 = plan.group_rows;
  const int step = plan.own_groups ? 1 : slots * plan.parts;     // the blocks of a group walk its rows side by side
  for (int set = first_set; set < sets; set += stride_set) {
    const int group = plan.own_groups ? set * slots + slot : set;
    const bool group_live = group < plan.groups;
    float g[K][8];
    if constexpr (GROUP) {
      const float* row_g = reinterpret_cast<const float*>(p.gate) + (int64_t)(group_live ? group : 0) * p.ldgate;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        load8<DT_F32>(row_g, c[k], C, g[k]);
        if (p.sigmoid) {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[k][j] = sigmoid_f<true>(g[k][j]).a;
        }
      }
    }
    // a row that is not there has no channels: zeros are read and nothing is written for it
    auto row_of = [&](int rr, int64_t* r) {
      const int in_group = plan.own_groups ? rr : rr + slot;
      const bool live = (WIDE || group_live) && in_group < row1;
      *r = live ? (int64_t)group * plan.group_rows + in_group : 0;
      return live ? C : 0;
    };
    auto work = [&](RowIn<DT, K>& in, int rr) __attribute__((always_inline)) {
      int64_t r;
      const int Cr = row_of(rr, &r);
      float up[K][8], h[K][8], v[K][8];
#pragma unroll
      for (int k = 0; k < K; ++k) unpack8<DT>(in.dh[k], up[k]);
      float s[3] = {0.f, 0.f, 0.f};
      float rs = 1.f, m_d = 0.f;
      if (has_y) {
#pragma unroll
        for (int k = 0; k < K; ++k) unpack8<DT>(in.y[k], v[k]);
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
      }
      if (has_dz) {
#pragma unroll
        for (int k = 0; k < K; ++k) unpack8<DT>(in.h[k], h[k]);
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) h[k][j] = 0.f;
      }
      if (!KEPT) get_pre();
      if (has_dz || p.post_gamma) {
        // both norms' statistics and what the first gradient needs come from the same sums
        if constexpr (LAYER) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            float dz[8];
            if (has_dz) unpack8<DT>(in.dz[k], dz);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              s[0] += h[k][j];
              s[1] += v[k][j];
              if (has_dz) s[2] += dz[j] * qw[k][j];
            }
          }
          row_sums<LPR, WIDE, 3>(s, red, turn);
          const float mean_h = s[0] * inv_c, mean_y = p.post_gamma ? s[1] * inv_c : 0.f;
          m_d = s[2] * inv_c;
          centre<K, ODD>(h, c, Cr, mean_h);
          centre<K, ODD>(v, c, Cr, mean_y);
          s[0] = s[1] = s[2] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float dz[8];
          if (has_dz) unpack8<DT>(in.dz[k], dz);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            s[0] += h[k][j] * h[k][j];
            s[1] += v[k][j] * v[k][j];
            if (has_dz) s[2] += dz[j] * qw[k][j] * h[k][j];
          }
        }
        row_sums<LPR, WIDE, 3>(s, red, turn);
        if (p.post_gamma) rs = 1.f / sqrtf(s[1] * inv_c + p.eps);
      }
      if (has_dz) {
        const float rh = 1.f / sqrtf(s[0] * inv_c + p.eps), m_dot = s[2] * rh * inv_c;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          float dz[8];
          unpack8<DT>(in.dz[k], dz);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float hat = h[k][j] * rh;
            const float d = LAYER ? dz[j] * qw[k][j] - m_d : dz[j] * qw[k][j];
            up[k][j] += rh * (d - hat * m_dot);
            acc[0][k][j] += dz[j] * hat;
            if constexpr (LAYER) acc[2][k][j] += dz[j];
          }
        }
      }
#pragma unroll
      for (int k = 0; k < K; ++k) store_row<DT, NT, ODD>(p.dx, r * C, c[k], Cr, up[k]);
      if (!has_y) return;
      if (!KEPT) get_post();
      float t[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float a[8], dg[8];
        if constexpr (!GROUP) {
          if (element) unpack8<DT>(in.gate[k], a);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // (channels past the end: gamma is zero, so they add nothing to the row's sums; their own are not stored)
          const float u = p.scale * up[k][j];
          const float hat = v[k][j] * rs;
          const float n = LAYER ? hat * pw[k][j] + pb[k][j] : hat * pw[k][j];
          float dn = u;
          dg[j] = u * n;
          if constexpr (GROUP) {
            dn *= g[k][j];
            acc[GATE][k][j] += dg[j];
          } else if (element) {
            if (p.sigmoid) {
              const Sigmoid sg = sigmoid_f<DT == DT_F32>(a[j]);
              a[j] = sg.a;
              dg[j] *= sg.slope;
            }
            dn *= a[j];
          }
          acc[1][k][j] += dn * hat;
          if constexpr (LAYER) acc[3][k][j] += dn;
          v[k][j] = hat;
          up[k][j] = dn * pw[k][j];
          t[0] += up[k][j] * hat;
          t[1] += up[k][j];
        }
        if constexpr (!GROUP) {
          if (element) store_row<DT, NT, ODD>(p.dgate, r * C, c[k], Cr, dg);
        }
      }
      if (p.post_gamma) {
        row_sums<LPR, WIDE, LAYER ? 2 : 1>(t, red, turn);
        const float m_dot = t[0] * inv_c, m_t = LAYER ? t[1] * inv_c : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) up[k][j] = rs * (up[k][j] - m_t - v[k][j] * m_dot);
      }
#pragma unroll
      for (int k = 0; k < K; ++k) store_row<DT, NT, ODD>(p.dy, r * C, c[k], Cr, up[k]);
    };
    if constexpr (FULL) {
      // lanes past the row's end, slots past a group's last row or the last group
      const bool ragged = C != lanes * 8 || (!WIDE && (plan.own_groups || plan.group_rows % slots != 0));
      auto ask = [&](int rr, RowIn<DT, K>& to) __attribute__((always_inline)) {
        int64_t r;
        row_of(rr, &r);
        load_full<DT, K, NT, MODE>(to, p, r, at);
      };
      auto take = [&](RowIn<DT, K>& in, int rr) __attribute__((always_inline)) {
        if (ragged) {
          int64_t r;
          const bool keep = c[0] < row_of(rr, &r);
          drop<DT>(in.dh[0], keep);
          drop<DT>(in.dz[0], keep);
          drop<DT>(in.h[0], keep);
          drop<DT>(in.y[0], keep);
          if constexpr (MODE == FULL_ELEMENT) drop<DT>(in.gate[0], keep);
        }
        work(in, rr);
      };
      RowIn<DT, K> a, b;       // two rows under way, in registers of their own: copying one would wait for it
      if (row0 < row1) ask(row0, a);
      for (int rr = row0; rr < row1; rr += 2 * step) {
        ask(rr + step, b);
        take(a, rr);
        if (rr + step >= row1) break;
        ask(rr + 2 * step, a);
        take(b, rr + step);
      }
    } else {
      RowIn<DT, K> next;
      auto ask = [&](int rr) {
        if (rr >= row1) return;
        int64_t r;
        const bool live = row_of(rr, &r) > 0;
        load_row<DT, K, NT, LPR == 2>(next, p, r, live, at);
      };
      ask(row0);
      for (int rr = row0; rr < row1; rr += step) {
        RowIn<DT, K> in = next;
        ask(rr + step);                    // before anything waits for this row
        settle_row(in, p, at);
        work(in, rr);
      }
    }
    if (GROUP && plan.parts == 1) {
      // whole groups: the gate's gradient is complete here
      if (WIDE || plan.own_groups) {
        if (group_live) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            if (p.sigmoid) {
              load8<DT_F32>(reinterpret_cast<const float*>(p.gate) + (int64_t)group * p.ldgate, c[k], C, g[k]);
#pragma unroll
              for (int j = 0; j < 8; ++j) acc[GATE][k][j] *= sigmoid_f<true>(g[k][j]).slope;
            }
            store8<DT_F32>(reinterpret_cast<float*>(p.dgate) + (int64_t)group * C, c[k], C, acc[GATE][k]);
          }
        }
      } else if constexpr (!WIDE) {
        over_slots<LPR>(acc[GATE][0], join, [&](int col, double sum) {
          if (col >= C) return;
          if (p.sigmoid)
            sum *= sigmoid_f<true>(reinterpret_cast<const float*>(p.gate)[(int64_t)group * p.ldgate + col]).slope;
          reinterpret_cast<float*>(p.dgate)[(int64_t)group * C + col] = (float)sum;
        });
      }
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[GATE][k][j] = 0.f;
    }
  }
  // the block's row of partial sums
#pragma unroll
  for (int i = 0; i < SUMS; ++i) {
    float* to = part.row[GROUP && i == GATE ? 4 : i];
    if (!to) continue;
    to += (int64_t)blockIdx.x * C;
    if constexpr (WIDE) {
#pragma unroll
      for (int k = 0; k < K; ++k) store8<DT_F32>(to, c[k], C, acc[i][k]);
    } else {
      over_slots<LPR>(acc[i][0], join, [&](int col, double sum) {
        if (col < C) to[col] = (float)sum;
      });
    }
  }
}

// Sums the blocks' partial rows, in one launch.  The vectors' rows (all blocks') and a gate's (of one group, `parts`
// of them) are taken 32 columns a block in 32 slices; gates of few parts go a column a thread, 1024 a block, where
// slices would leave most of a block idle (256 groups of 4 parts, 2048 columns: 35 us in slices, 5 us this way).
struct Finish {
  const float* from[5];
  float* to[5];
  const float* gate;
  int64_t ldgate;
  int C, rows, parts, groups, sigmoid;
  int vector_blocks;      // blocks of the vectors; the gate's follow
};
constexpr int FEW_PARTS = 32;

// (a template so that every element type's file has its own)
template <int DT>
__global__ __launch_bounds__(1024) void finish_kernel(const Finish f) {
  __shared__ double join[32][33];
  const int cols = (f.C + 31) / 32;
  int b = (int)blockIdx.x, i = 4, group = 0, rows = f.parts, col;
  if (b < f.vector_blocks) {
    // the b / cols-th vector that is wanted
    int skip = b / cols;
    i = 0;
    while (f.to[i] == nullptr || skip-- > 0) ++i;
    b %= cols;
    rows = f.rows;
  } else {
    b -= f.vector_blocks;
    if (f.parts <= FEW_PARTS) {
      const int wide_cols = (f.C + 1023) / 1024;
      group = b / wide_cols;
      col = (b % wide_cols) * 1024 + (int)threadIdx.x;
      if (col >= f.C) return;
      const float* from = f.from[4] + (int64_t)group * f.parts * f.C + col;
      double sum = 0.;
#pragma unroll 4
      for (int r = 0; r < f.parts; ++r) sum += from[(int64_t)r * f.C];
      if (f.sigmoid) sum *= sigmoid_f<true>(f.gate[(int64_t)group * f.ldgate + col]).slope;
      f.to[4][(int64_t)group * f.C + col] = (float)sum;
      return;
    }
    group = b / cols;
    b %= cols;
  }
  col = b * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  double sum = 0.;
  if (col < f.C) {
    const float* from = f.from[i] + (int64_t)group * f.parts * f.C + col;
#pragma unroll 16
    for (int r = slice; r < rows; r += 32) sum += from[(int64_t)r * f.C];
  }
  join[slice][threadIdx.x & 31] = sum;
  __syncthreads();
  if (slice == 0 && col < f.C) {
    sum = 0.;
#pragma unroll
    for (int q = 0; q < 32; ++q) sum += join[q][threadIdx.x];
    if (i == 4 && f.sigmoid) sum *= sigmoid_f<true>(f.gate[(int64_t)group * f.ldgate + col]).slope;
    f.to[i][(int64_t)group * f.C + col] = (float)sum;
  }
}

// (lanes per row, wide, chunks per lane) by the row's length alone: eight channels a lane while that takes at most
// 512 threads, sixteen above.
#define DTF_ROW_SWITCH(C, ...)                                                                     \
  do {                                                                                             \
    if ((C) <= 16) { constexpr int LPR = 2, K = 1; constexpr bool WIDE = false; __VA_ARGS__; }      \
    else if ((C) <= 32) { constexpr int LPR = 4, K = 1; constexpr bool WIDE = false; __VA_ARGS__; } \
    else if ((C) <= 64) { constexpr int LPR = 8, K = 1; constexpr bool WIDE = false; __VA_ARGS__; } \
    else if ((C) <= 128) { constexpr int LPR = 16, K = 1; constexpr bool WIDE = false; __VA_ARGS__; } \
    else if ((C) <= 256) { constexpr int LPR = 32, K = 1; constexpr bool WIDE = false; __VA_ARGS__; } \
    else if ((C) <= 512) { constexpr int LPR = 64, K = 1; constexpr bool WIDE = false; __VA_ARGS__; } \
    else if ((C) <= 4096) { constexpr int LPR = 64, K = 1; constexpr bool WIDE = true; __VA_ARGS__; } \
    else { constexpr int LPR = 64, K = 2; constexpr bool WIDE = true; __VA_ARGS__; }                \
  } while (0)

template <int DT>
void launch_fwd(const ResidualNormParams& p, hipStream_t s) {
  const int threads = p.C <= 512 ? 256 : wide_threads(p.C);
  const int nt = big(p, 4), blocks = fwd_blocks(p, nt);
  const int mode = !full_rows(p) ? (int)ANY : p.gate_mode == GATE_GROUP ? (int)FULL_GROUP :
                   p.gate_mode == GATE_ELEMENT ? (int)FULL_ELEMENT : (int)FULL_PLAIN;
#define DTF_FWD(LAYER, MODE)                                                                                    \
  DTF_ROW_SWITCH(p.C, if (nt) {                                                                                    \
    hipLaunchKernelGGL((fwd_kernel<DT, LPR, WIDE, K, LAYER, K == 1 ? MODE : (int)ANY, true>), dim3(blocks),       \
                       dim3(threads), 0, s, p);                                                                   \
  } else {                                                                                                        \
    hipLaunchKernelGGL((fwd_kernel<DT, LPR, WIDE, K, LAYER, K == 1 ? MODE : (int)ANY, false>), dim3(blocks),      \
                       dim3(threads), 0, s, p);                                                                   \
  })
#define DTF_FWD_LAYER(MODE)                       \
  do {                                            \
    if (p.layer) { DTF_FWD(true, MODE); } else { DTF_FWD(false, MODE); } \
  } while (0)
  switch (mode) {
    case FULL_PLAIN: DTF_FWD_LAYER(FULL_PLAIN); break;
    case FULL_GROUP: DTF_FWD_LAYER(FULL_GROUP); break;
    case FULL_ELEMENT: DTF_FWD_LAYER(FULL_ELEMENT); break;
    default: DTF_FWD_LAYER(ANY); break;
  }
#undef DTF_FWD_LAYER
#undef DTF_FWD
}

template <int DT>
void launch_bwd(const ResidualNormParams& p, hipStream_t s) {
  const bool full = full_rows(p) && p.dz && p.dh;
  const BwdPlan plan = plan_bwd(p, full);
  const int threads = p.C <= 512 ? 256 : wide_threads(p.C);
  float* to[5] = {p.dpre_gamma, p.dpost_gamma, p.dpre_beta, p.dpost_beta, nullptr};
  if (p.gate_mode == GATE_GROUP && plan.parts > 1) to[4] = reinterpret_cast<float*>(p.dgate);
  Partials part;
  Finish f;
  int vectors = 0;
  for (int i = 0; i < 5; ++i) {
    part.row[i] = to[i] ? p.ws + (size_t)i * plan.blocks * p.C : nullptr;
    f.from[i] = part.row[i];
    f.to[i] = to[i];
    vectors += i < 4 && to[i];
  }
  const bool grouped = p.gate_mode == GATE_GROUP;
  const int mode = !full ? (grouped ? (int)ANY_GROUP : (int)ANY) :
                   grouped ? (int)FULL_GROUP : p.gate_mode == GATE_ELEMENT ? (int)FULL_ELEMENT : (int)FULL_PLAIN;
#define DTF_BWD(LAYER, MODE)                                                                                    \
  DTF_ROW_SWITCH(p.C, constexpr int M = K == 1 || MODE < FULL_PLAIN ? MODE : (int)ANY; if (plan.nt) {               \
    hipLaunchKernelGGL((bwd_kernel<DT, LPR, WIDE, K, LAYER, M, true>), dim3(plan.blocks), dim3(threads), 0, s, p,  \
                       plan, part);                                                                               \
  } else {                                                                                                        \
    hipLaunchKernelGGL((bwd_kernel<DT, LPR, WIDE, K, LAYER, M, false>), dim3(plan.blocks), dim3(threads), 0, s, p, \
                       plan, part);                                                                               \
  })
#define DTF_BWD_LAYER(MODE)                       \
  do {                                            \
    if (p.layer) { DTF_BWD(true, MODE); } else { DTF_BWD(false, MODE); } \
  } while (0)
  switch (mode) {
    case FULL_PLAIN: DTF_BWD_LAYER(FULL_PLAIN); break;
    case FULL_GROUP: DTF_BWD_LAYER(FULL_GROUP); break;
    case FULL_ELEMENT: DTF_BWD_LAYER(FULL_ELEMENT); break;
    case ANY_GROUP: DTF_BWD_LAYER(ANY_GROUP); break;
    default: DTF_BWD_LAYER(ANY); break;
  }
#undef DTF_BWD_LAYER
#undef DTF_BWD
  if (!vectors && !to[4]) return;
  f.gate = reinterpret_cast<const float*>(p.gate);
  f.ldgate = p.ldgate;
  f.C = p.C;
  f.rows = plan.blocks;
  f.parts = plan.parts;
  f.groups = plan.groups;
  f.sigmoid = p.sigmoid;
  f.vector_blocks = vectors * ((p.C + 31) / 32);
  const int gates = to[4] ? plan.groups * (plan.parts <= FEW_PARTS ? (p.C + 1023) / 1024 : (p.C + 31) / 32) : 0;
  hipLaunchKernelGGL(finish_kernel<DT>, dim3(f.vector_blocks + gates), dim3(1024), 0, s, f);
}

}  // namespace rn
