// Dropout on [n, c] activations: y = kept ? x / (1 - p) : 0.  The mask comes from a counter-based generator (rowops.h)
// and is never stored: the backward pass is the same call on the gradient, with the same seed and offset.
#include "rowops.h"

namespace m3d {

constexpr int kDropThreads = 256;

// A workgroup owns kDropThreads * U consecutive pieces (16 bytes) of the logical [n][c] tensor; a piece is (row, piece of
// the row), the division by the pieces of a row is a multiplication (magic, shift: exact below 2^31 pieces).  WHOLE: no row
// ends inside a piece.
// Bound by HBM: the generator's 7 rounds are 14 widening products for 4 values, which the memory time covers (273080 x 96
// f32 34.2 us, 6.1 TB/s; 16384 x 4096 bf16 44.9 us, 6.0 TB/s).
template <typename T, int U, bool WHOLE>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const T* __restrict__ x, int64_t ldx, int c, int64_t row0,
                                                               uint32_t total, uint32_t per_row, uint32_t magic,
                                                               int shift, DropArgs d, T* __restrict__ y) {
  constexpr int V = kPiece<T>;
  const DropKey key = drop_key(d);
  const uint32_t base = blockIdx.x * (kDropThreads * U) + threadIdx.x;
  Piece<T, V> in[U];
  uint32_t row[U];
  int col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t t = base + u * kDropThreads;
    row[u] = (__umulhi(magic, t) + t) >> shift;
    col[u] = (int)(t - row[u] * per_row) * V;
    const T* p = x + (row0 + row[u]) * ldx + col[u];
    const int left = t < total ? c - col[u] : 0;
    if constexpr (WHOLE) {
      if (left > 0) in[u].load_stream(p);
    } else if (left >= V) {
      in[u].load(p);
    } else {
      in[u].load_some(p, 0, left);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t t = base + u * kDropThreads;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = in[u].get(i);
    if (d.on) drop<V>(v, col[u], (uint32_t)(row0 + row[u]), key, d.last, d.scale);
#pragma unroll
    for (int i = 0; i < V; ++i) in[u].set(i, v[i]);
    T* p = y + (row0 + row[u]) * c + col[u];
    const int left = t < total ? c - col[u] : 0;
    if (left >= V) in[u].store(p);
    else if constexpr (!WHOLE) in[u].store_some(p, 0, left);
  }
}

template <typename T, int U, bool WHOLE>
static int dropout_launch(const T* x, int64_t ldx, int64_t n, int c, const DropArgs& d, T* y, hipStream_t stream) {
  constexpr int V = kPiece<T>;
  const uint32_t per_row = (uint32_t)cdiv(c, V);
  int shift = 0;
  while ((1ull << shift) < per_row) ++shift;
  const uint32_t magic = (uint32_t)((((1ull << shift) - per_row) << 32) / per_row + 1);
  // piece indices stay below 2^31 - (one workgroup): longer tensors take several launches
  const int64_t rows_max = ((int64_t)0x7fff0000) / per_row;
  for (int64_t r0 = 0; r0 < n; r0 += rows_max) {
    const int64_t rows = n - r0 < rows_max ? n - r0 : rows_max;
    const uint32_t total = (uint32_t)(rows * per_row);
    hipLaunchKernelGGL((dropout_kernel<T, U, WHOLE>), dim3((unsigned)cdiv(total, kDropThreads * U)), dim3(kDropThreads), 0,
                       stream, x, ldx, c, r0, total, per_row, magic, shift, d, y);
    M3D_LAUNCH_CHECK();
  }
  return M3D_OK;
}

// Pieces a thread: two of whole 16-bit pieces (16384 x 4096 bf16, the call on x and on the gradient: 93.8 us, with one
// 94.6), one otherwise (273080 x 96 f32: 34.2 us, with two 34.9, with four 34.4; 75401 x 333 f16, whose rows end inside a
// piece: 23.2, with two 25.4, with four 26.5).
template <typename T>
static int dropout_typed(const void* x, int64_t ldx, int64_t n, int c, const DropArgs& d, void* y, hipStream_t stream) {
  const T* from = static_cast<const T*>(x);
  if (c % kPiece<T> == 0)
    return dropout_launch<T, sizeof(T) == 2 ? 2 : 1, true>(from, ldx, n, c, d, static_cast<T*>(y), stream);
  return dropout_launch<T, 1, false>(from, ldx, n, c, d, static_cast<T*>(y), stream);
}

// One thread: hands a call its (seed, offset) and moves the state on.
__global__ void dropout_next_kernel(int64_t* state, int64_t step, int64_t* used) {
  used[0] = state[0];
  used[1] = state[1];
  state[1] += step;
}

}  // namespace m3d

using namespace m3d;

extern "C" int m3d_dropout(const void* d_x, int64_t ldx, int type, int64_t n, int c, double p, uint64_t seed,
                           uint64_t offset, const int64_t* d_state, void* d_y, void* stream_) {
  const char* who = "m3d_dropout";
  M3D_CHECK_ARG(type_ok(type), "%s: unknown element type %d", who, type);
  M3D_CHECK_ARG(n >= 0 && n < (int64_t)1 << 32 && c >= 1 && c < 1 << 30, "%s: %lld rows of %d channels are not supported",
                who, (long long)n, c);
  DropArgs d;
  if (int rc = drop_args(who, p, seed, offset, d_state, &d)) return rc;
  if (n == 0) return M3D_OK;
  M3D_CHECK_ARG(d_x && d_y, "%s: null pointer", who);
  M3D_CHECK_ARG(ldx >= c || n == 1, "%s: row stride %lld is smaller than the %d channels", who, (long long)ldx, c);
  M3D_CHECK_ARG((((uintptr_t)d_x | (uintptr_t)d_y) & (type_bytes(type) - 1)) == 0, "%s: misaligned pointer", who);
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (type == M3D_TYPE_F32) return dropout_typed<float>(d_x, ldx, n, c, d, d_y, stream);
  if (type == M3D_TYPE_BF16) return dropout_typed<bf16_t>(d_x, ldx, n, c, d, d_y, stream);
  return dropout_typed<f16_t>(d_x, ldx, n, c, d, d_y, stream);
}

extern "C" int m3d_dropout_next(int64_t* d_state, int64_t step, int64_t* d_used, void* stream) {
  const char* who = "m3d_dropout_next";
  M3D_CHECK_ARG(d_state && d_used, "%s: null pointer", who);
  M3D_CHECK_ARG((((uintptr_t)d_state | (uintptr_t)d_used) & 7) == 0, "%s: pointers must be 8-byte aligned", who);
  hipLaunchKernelGGL(dropout_next_kernel, dim3(1), dim3(1), 0, static_cast<hipStream_t>(stream), d_state, step, d_used);
  M3D_LAUNCH_CHECK();
  return M3D_OK;
}
