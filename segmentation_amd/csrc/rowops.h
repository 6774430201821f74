// What the row-wise operators on [n, c] activations share (layer_norm.hip, dropout.hip): element types, 16-byte pieces
// of a row at any alignment, sums over the lanes that hold a row, and the generator behind dropout masks.
#pragma once
#include "common.h"

namespace m3d {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct TypeCode;
template <> struct TypeCode<float> { static constexpr int value = M3D_TYPE_F32; };
template <> struct TypeCode<bf16_t> { static constexpr int value = M3D_TYPE_BF16; };
template <> struct TypeCode<f16_t> { static constexpr int value = M3D_TYPE_F16; };

static inline bool type_ok(int t) { return t == M3D_TYPE_F32 || t == M3D_TYPE_BF16 || t == M3D_TYPE_F16; }
static inline size_t type_bytes(int t) { return t == M3D_TYPE_F32 ? 4 : 2; }

// V consecutive channels of a row.  The vector types claim no more than the element's alignment: the compiler still
// emits 16-byte accesses (gfx950 takes them at any address), so that odd channel counts, row strides and sliced
// tensors run through the same code as aligned ones.
template <typename T, int V>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef T uvec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  vec v;
  __device__ __forceinline__ void load(const T* __restrict__ p) { v = *reinterpret_cast<const uvec*>(p); }
  // Activations that a kernel reads once: marked as a stream, so that they do not push its outputs out of the caches.
  // Forward of 8192 x 8192 bf16 50.6 -> 44.5 us; forward and backward behind the add 75401 x 256 f32 136 -> 127, 16384 x
  // 4096 bf16 233 -> 229; a layer norm whose backward pass follows at once and found its input in the cache before loses
  // (273080 x 96 f32 98.6 -> 101).  Marking the forward or the backward pass alone is slower than both (110, 108).
  // What shares a line with another load is loaded plainly: the two halves of a 32-byte piece (30001 x 768 bf16 on an f32
  // stream 115 us, marked 126), and, by the callers' choice, rows that are no multiple of a piece (1 M x 65 f32 layer norm
  // behind the add 4.2 TB/s, marked 3.7).
  __device__ __forceinline__ void load_stream(const T* __restrict__ p) {
    if constexpr (V * sizeof(T) == 16) v = (vec)__builtin_nontemporal_load(reinterpret_cast<const uvec*>(p));
    else load(p);
  }
  __device__ __forceinline__ void store(T* __restrict__ p) const { *reinterpret_cast<uvec*>(p) = v; }
  // positions [from, to) only; the others load as zero
  __device__ __forceinline__ void load_some(const T* __restrict__ p, int from, int to) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i >= from && i < to ? p[i] : (T)0.f;
  }
  __device__ __forceinline__ void store_some(T* __restrict__ p, int from, int to) const {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i >= from && i < to) p[i] = v[i];
  }
  __device__ __forceinline__ float get(int i) const { return (float)v[i]; }
  __device__ __forceinline__ void set(int i, float f) { v[i] = (T)f; }
};

// Where a lane's piece lies in its row of c channels: channels col .. col + V - 1, of which the first `skip` belong to
// the lane before (the last piece of a row that is no multiple of V is moved back so that it ends with the row) or,
// with skip = V, all do (a lane without a piece of its own).  Only a row of fewer than V channels has `count` < V.
struct Place {
  int col, skip, count;
};

template <int V>
__device__ __forceinline__ Place place_of(int piece, int c) {
  const int whole = c / V;
  if (piece < whole) return {piece * V, 0, V};
  if (c < V) return {0, piece == 0 ? 0 : V, c};
  return {c - V, piece == whole ? V - c % V : V, V};  // c % V == 0: V, nothing is left for this lane
}

// channels per piece: 16 bytes of the activations' type
template <typename T> constexpr int kPiece = 16 / (int)sizeof(T);

// V parameters (weight or bias, f32 or the 16-bit types) as f32; p == nullptr: `none`
template <int V>
__device__ __forceinline__ void load_params(const void* p, int type, const Place& at, float none, float* out) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = none;
  } else if (type == M3D_TYPE_F32) {
    Piece<float, V> q;
    if (at.count == V) q.load(static_cast<const float*>(p) + at.col);
    else q.load_some(static_cast<const float*>(p), 0, at.count);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = q.get(i);
  } else if (type == M3D_TYPE_BF16) {
    Piece<bf16_t, V> q;
    if (at.count == V) q.load(static_cast<const bf16_t*>(p) + at.col);
    else q.load_some(static_cast<const bf16_t*>(p), 0, at.count);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = q.get(i);
  } else {
    Piece<f16_t, V> q;
    if (at.count == V) q.load(static_cast<const f16_t*>(p) + at.col);
    else q.load_some(static_cast<const f16_t*>(p), 0, at.count);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = q.get(i);
  }
}

// ---------------------------------------------------------------- sums over groups of lanes
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
  return v + __builtin_bit_cast(float, o);
}

// Sums over aligned groups of g lanes (g a power of two, 1..64, the same in every lane); every lane gets them.  The
// four steps inside 16 lanes are lane permutations of the add itself, 16 and 32 are row and half swaps.  The sums go
// through a step together, so that two take little longer than one.
template <int NQ>
__device__ __forceinline__ void group_sum(float (&v)[NQ], int g) {
  if (g > 1)
#pragma unroll
    for (int q = 0; q < NQ; ++q) v[q] = dpp_add<0xB1>(v[q]);    // lane ^ 1
  if (g > 2)
#pragma unroll
    for (int q = 0; q < NQ; ++q) v[q] = dpp_add<0x4E>(v[q]);    // lane ^ 2
  if (g > 4)
#pragma unroll
    for (int q = 0; q < NQ; ++q) v[q] = dpp_add<0x141>(v[q]);   // mirror inside 8 lanes (quads are equal by now)
  if (g > 8)
#pragma unroll
    for (int q = 0; q < NQ; ++q) v[q] = dpp_add<0x140>(v[q]);   // mirror inside 16 lanes
  if (g > 16)
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int b = __builtin_bit_cast(int, v[q]);
      const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
      const unsigned lo = s[0], hi = s[1];
      v[q] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    }
  if (g > 32)
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int b = __builtin_bit_cast(int, v[q]);
      const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
      const unsigned lo = s[0], hi = s[1];
      v[q] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    }
}

// ---------------------------------------------------------------- dropout masks
// Philox 4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with 7 rounds, the
// fewest that pass its authors' whole test battery (with 10, 16384 x 4096 bf16 values take 58 us instead of 48.6: the
// products, not the memory, bound them).  A block of four 32-bit words belongs to four consecutive channels
// of a row: counter = (channel / 4, row, offset low, offset high), key = seed.  A value is kept where its word is at
// least p * 2^32, so the mask is a function of (seed, offset, row, channel) alone, whatever the type, stride or kernel.
struct DropArgs {
  const int64_t* state;  // device (seed, offset) or nullptr; `offset` is added to the state's
  uint64_t seed, offset;
  uint32_t last;         // the largest word that is dropped
  float scale;           // 1 / (1 - p)
  int on;                // 0: nothing is dropped
};

struct DropKey {
  uint32_t k0, k1, o0, o1;
};

__device__ __forceinline__ DropKey drop_key(const DropArgs& a) {
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state) {
    seed = (uint64_t)a.state[0];
    offset += (uint64_t)a.state[1];
  }
  return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}

__device__ __forceinline__ void philox7(uint32_t chunk, uint32_t row, const DropKey& key, uint32_t (&w)[4]) {
  uint32_t c0 = chunk, c1 = row, c2 = key.o0, c3 = key.o1, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// v[i] = kept ? v[i] * scale : 0 for V channels from `col` (a multiple of 4).  The product is rounded by itself (no
// contraction into a following add): dropout alone and dropout in front of an add give the same values.
template <int V>
__device__ __forceinline__ void drop(float* v, int col, uint32_t row, const DropKey& key, uint32_t last, float scale) {
#pragma clang fp contract(off)
#pragma unroll
  for (int q = 0; q < V; q += 4) {
    uint32_t w[4];
    philox7((uint32_t)(col + q) >> 2, row, key, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float kept = v[q + i] * scale;
      v[q + i] = w[i] > last ? kept : 0.f;
    }
  }
}

// drop() for a piece that starts anywhere: the words of the blocks it touches, moved into place.
template <int V>
__device__ __forceinline__ void drop_unaligned(float* v, int col, uint32_t row, const DropKey& key, uint32_t last,
                                               float scale) {
#pragma clang fp contract(off)
  uint32_t w[V + 4];
#pragma unroll
  for (int q = 0; q < V + 4; q += 4) {
    uint32_t b[4];
    philox7((uint32_t)(col + q) >> 2, row, key, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[q + i] = b[i];
  }
  const int by = col & 3;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t word = by == 0 ? w[i] : by == 1 ? w[i + 1] : by == 2 ? w[i + 2] : w[i + 3];
    const float kept = v[i] * scale;
    v[i] = word > last ? kept : 0.f;
  }
}

// Host: p -> DropArgs.  p in [0, 1]; values are dropped with probability round(p * 2^32) / 2^32.
static inline int drop_args(const char* who, double p, uint64_t seed, uint64_t offset, const int64_t* state,
                            DropArgs* out) {
  M3D_CHECK_ARG(p >= 0.0 && p <= 1.0, "%s: dropout probability %g is not in [0, 1]", who, p);
  M3D_CHECK_ARG(((uintptr_t)state & 7) == 0, "%s: the generator state must be 8-byte aligned", who);
  const double words = p * 4294967296.0;
  const uint64_t count = (uint64_t)__builtin_rint(words);  // words 0 .. count - 1 are dropped
  out->state = state;
  out->seed = seed;
  out->offset = offset;
  out->on = count > 0;
  out->last = count > 0 ? (uint32_t)(count - 1) : 0;
  out->scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  return M3D_OK;
}

}  // namespace m3d
