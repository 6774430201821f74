// Layer norm over the channels of every row of [n, c] activations, forward and backward, alone and behind the residual
// add of a block:
//   alone:  y = (x - mean) * rstd * weight + bias,  mean and rstd = 1 / sqrt(var + eps) of the row
//   add:    h = residual + dropout(x) (rounded to the stream's type), y = layer norm of h as it is held
//   backward, with hat = (x - mean) * rstd and g = dy * weight:
//           dx = rstd * (g - mean(g) - hat * mean(g * hat)) [+ dh, and dropout's mask for x's own gradient]
//           dweight = sum over rows of dy * hat,  dbias = sum over rows of dy
//
// A row is held by a group of lanes in registers (K pieces of 16 bytes a lane), so that every input is read once:
// the mean, the squared deviations from it and the output come from the same registers.  Groups inside a wave add by
// lane permutations, wider rows take a group of several waves that add through LDS.  All sums are f32.
// The column sums of the backward pass stay in registers over all rows of a workgroup, are joined inside it, written as
// one partial row per workgroup and added up by a second launch in a fixed order (no atomics: run-to-run identical).
#include "rowops.h"

namespace m3d {

struct LnArgs {
  const void* in;        // forward: x.  backward: the norm's input (x, or h of the add)
  int64_t ld_in;
  const void* residual;  // forward of the add
  int64_t ld_res;
  const void* dy;        // backward
  int64_t ld_dy;
  const void* dh;        // backward of the add, or nullptr
  int64_t ld_dh;
  const void* weight;
  const void* bias;
  int wtype;
  int64_t n;
  int c, lg;             // 1 << lg lanes hold a row
  float inv_c, eps;
  void* y;               // forward outputs
  void* h;               // or nullptr
  float* mean;           // forward: written, backward: read
  float* rstd;
  void* dx;              // backward outputs, either may be nullptr for the add
  void* dres;
  float* partial;        // [workgroups][2][c] or nullptr
  int64_t tiles;
  DropArgs drop;
};

// Sums over the 1 << lg lanes of a row.  Rows wider than a wave: wave sums go through LDS, in wave order; the two
// slots take turns, so one barrier per sum is enough (a wave that writes a slot again has passed the barrier behind
// which every wave had read it).  Every wave of the workgroup must make the same calls.
template <int THREADS, int NQ>
struct RowSum {
  float (*red)[THREADS / 64][NQ];
  int turn = 0;
  __device__ __forceinline__ void operator()(float (&v)[NQ], int lg) {
    const int g = 1 << lg;
#pragma unroll
    for (int q = 0; q < NQ; ++q) v[q] = group_sum(v[q], g < 64 ? g : 64);
    if (lg > 6) {
      const int wave = threadIdx.x >> 6, waves = g >> 6, first = wave & ~(waves - 1);
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int q = 0; q < NQ; ++q) red[turn][wave][q] = v[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NQ; ++q) v[q] = 0.f;
      for (int w = 0; w < waves; ++w)
#pragma unroll
        for (int q = 0; q < NQ; ++q) v[q] += red[turn][first + w][q];
      turn ^= 1;
    }
  }
};

template <typename TX, typename TR, int K, bool ADD, int THREADS>
__global__ __launch_bounds__(THREADS) void ln_fwd_kernel(LnArgs a) {
  constexpr int V = kPiece<TX>;
  __shared__ float red[2][THREADS / 64][1];
  RowSum<THREADS, 1> row_sum{red};
  const int g = 1 << a.lg, lane = threadIdx.x & (g - 1), slot = threadIdx.x >> a.lg, rows = THREADS >> a.lg;
  const bool ragged = a.c % V != 0;
  DropKey key = {};
  if (ADD && a.drop.on) key = drop_key(a.drop);
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (lane + k * g) * V;
    load_params<V>(a.weight, a.wtype, col, a.c - col, 1.f, w[k]);
    load_params<V>(a.bias, a.wtype, col, a.c - col, 0.f, b[k]);
  }
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t row = tile * rows + slot;
    const int c = row < a.n ? a.c : 0;  // rows behind the last one load and store nothing
    float v[K][V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * g) * V;
      Piece<TX, V> x;
      x.load(static_cast<const TX*>(a.in) + row * a.ld_in + col, c - col);
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = x.get(i);
      if constexpr (ADD) {
        Piece<TR, V> r;
        r.load(static_cast<const TR*>(a.residual) + row * a.ld_res + col, c - col);
        if (a.drop.on) drop<V>(v[k], col, (uint32_t)row, key, a.drop.last, a.drop.scale);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          r.set(i, r.get(i) + v[k][i]);
          v[k][i] = r.get(i);
        }
        if (a.h) r.store(static_cast<TR*>(a.h) + row * a.c + col, c - col);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += v[k][i];
    }
    row_sum(s, a.lg);
    const float mean = s[0] * a.inv_c;
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int left = c - (lane + k * g) * V;
      const float mu = left > 0 ? mean : 0.f;  // pieces behind the row's end: all zero, and so is their deviation
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] -= mu;
        if (ragged && i >= left) v[k][i] = 0.f;
        s[0] += v[k][i] * v[k][i];
      }
    }
    row_sum(s, a.lg);
    const float rstd = 1.f / __builtin_sqrtf(s[0] * a.inv_c + a.eps);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * g) * V;
      Piece<TX, V> y;
#pragma unroll
      for (int i = 0; i < V; ++i) y.set(i, v[k][i] * rstd * w[k][i] + b[k][i]);
      y.store(static_cast<TX*>(a.y) + row * a.c + col, c - col);
    }
    if (lane == 0 && row < a.n) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename TX, typename TR, int K, bool ADD, int THREADS>
__global__ __launch_bounds__(THREADS) void ln_bwd_kernel(LnArgs a) {
  constexpr int V = kPiece<TX>;
  __shared__ float red[2][THREADS / 64][2];
  RowSum<THREADS, 2> row_sum{red};
  const int g = 1 << a.lg, lane = threadIdx.x & (g - 1), slot = threadIdx.x >> a.lg, rows = THREADS >> a.lg;
  DropKey key = {};
  if (ADD && a.drop.on) key = drop_key(a.drop);
  float w[K][V], dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (lane + k * g) * V;
    load_params<V>(a.weight, a.wtype, col, a.c - col, 1.f, w[k]);
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  }
  for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
    const int64_t row = tile * rows + slot;
    const int c = row < a.n ? a.c : 0;
    const float mean = row < a.n ? a.mean[row] : 0.f, rstd = row < a.n ? a.rstd[row] : 0.f;
    Piece<TR, V> x[K], dh[K];
    Piece<TX, V> dy[K];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * g) * V;
      x[k].load(static_cast<const TR*>(a.in) + row * a.ld_in + col, c - col);
      dy[k].load(static_cast<const TX*>(a.dy) + row * a.ld_dy + col, c - col);
      if constexpr (ADD) dh[k].load(static_cast<const TR*>(a.dh) + row * a.ld_dh + col, a.dh ? c - col : 0);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {  // positions behind the row's end have dy = 0 and add nothing
        const float hat = (x[k].get(i) - mean) * rstd, d = dy[k].get(i), gw = d * w[k][i];
        dw[k][i] += d * hat;
        db[k][i] += d;
        s[0] += gw;
        s[1] += gw * hat;
      }
    row_sum(s, a.lg);
    const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * g) * V;
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float hat = (x[k].get(i) - mean) * rstd, gw = dy[k].get(i) * w[k][i];
        v[i] = (gw - m0 - hat * m1) * rstd;
        if constexpr (ADD) v[i] += dh[k].get(i);
      }
      if constexpr (ADD) {
        Piece<TR, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.set(i, v[i]);
        if (a.dres) out.store(static_cast<TR*>(a.dres) + row * a.c + col, c - col);
        if (a.drop.on) drop<V>(v, col, (uint32_t)row, key, a.drop.last, a.drop.scale);
      }
      Piece<TX, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) out.set(i, v[i]);
      if (a.dx) out.store(static_cast<TX*>(a.dx) + row * a.c + col, c - col);
    }
  }
  if (a.partial == nullptr) return;
  // The groups of a workgroup that hold the same channels are joined: lanes of a wave by shuffles, waves through LDS in
  // wave order (a group of several waves owns its channels alone within its slot).
  for (int o = g; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dw[k][i] += __shfl_xor(dw[k][i], o);
        db[k][i] += __shfl_xor(db[k][i], o);
      }
  const int waves = g > 64 ? g >> 6 : 1, slots = (THREADS / 64) / waves;  // slots: partial sums per channel
  const int me = (threadIdx.x >> 6) / waves;
  extern __shared__ float join[];  // [slots - 1][c]
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float* out = a.partial + ((int64_t)blockIdx.x * 2 + q) * a.c;
    const bool mine = (int)(threadIdx.x & 63) < g;
    if (q) __syncthreads();
    if (me > 0 && mine)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int col = (lane + k * g) * V + i;
          if (col < a.c) join[(me - 1) * a.c + col] = q ? db[k][i] : dw[k][i];
        }
    __syncthreads();
    if (me == 0 && mine)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int col = (lane + k * g) * V;
        Piece<float, V> sum;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float t = q ? db[k][i] : dw[k][i];
          if (col + i < a.c)
            for (int m = 0; m + 1 < slots; ++m) t += join[m * a.c + col + i];
          sum.set(i, t);
        }
        sum.store(out + col, a.c - col);
      }
  }
}

// dweight and dbias from the partial rows, in f64 and in a fixed order: a workgroup owns 32 columns of the 2 * c, each of
// its 32 row groups adds every 32nd partial row, and the group sums are added in group order.
__global__ __launch_bounds__(1024) void ln_columns_kernel(const float* __restrict__ partial, int blocks, int c, int wtype,
                                                          void* dweight, void* dbias) {
  __shared__ double red[32][33];
  const int e = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + e;
  double s = 0.0;
  if (col < 2 * c)
    for (int r = grp; r < blocks; r += 32) s += (double)partial[(int64_t)r * 2 * c + col];
  red[grp][e] = s;
  __syncthreads();
  if (grp == 0 && col < 2 * c) {
    double t = 0.0;
    for (int r = 0; r < 32; ++r) t += red[r][e];
    void* to = col < c ? dweight : dbias;
    const int at = col < c ? col : col - c;
    if (to == nullptr) return;
    if (wtype == M3D_TYPE_F32) static_cast<float*>(to)[at] = (float)t;
    else if (wtype == M3D_TYPE_BF16) static_cast<bf16_t*>(to)[at] = (bf16_t)(float)t;
    else static_cast<f16_t*>(to)[at] = (f16_t)(float)t;
  }
}

// ---------------------------------------------------------------- launch shapes
constexpr int kLnMaxChannels = 16384;

struct LnShape {
  int lg, k, threads;
};

// Lanes and pieces a lane for a row of `pieces` 16-byte pieces: the (lanes, K) that leave the fewest places empty.
static LnShape ln_shape(int pieces, int k_max) {
  LnShape best = {0, 0, 0};
  int waste = 0;
  for (int lg = 0; lg <= 10; ++lg) {
    const int g = 1 << lg, k = (int)cdiv(pieces, g);
    if (k > k_max || (g < 8 && g < pieces)) continue;
    if (best.k == 0 || g * k < waste) {
      best = {lg, k, lg > 8 ? 1024 : 256};
      waste = g * k;
    }
  }
  return best;
}

static int64_t ln_blocks(int64_t tiles) { return tiles < 2048 ? tiles : 2048; }
static int64_t ln_bwd_blocks(int64_t tiles) { return tiles < 1024 ? tiles : 1024; }

template <typename TX, typename TR, bool ADD, bool BWD, int K, int THREADS>
static int ln_launch_k(LnArgs& a, int64_t blocks, size_t lds, hipStream_t stream) {
  if constexpr (BWD)
    hipLaunchKernelGGL((ln_bwd_kernel<TX, TR, K, ADD, THREADS>), dim3((unsigned)blocks), dim3(THREADS), lds, stream, a);
  else
    hipLaunchKernelGGL((ln_fwd_kernel<TX, TR, K, ADD, THREADS>), dim3((unsigned)blocks), dim3(THREADS), 0, stream, a);
  M3D_LAUNCH_CHECK();
  return M3D_OK;
}

template <typename TX, typename TR, bool ADD, bool BWD>
static int ln_launch(LnArgs& a, int64_t* out_blocks, hipStream_t stream) {
  const LnShape s = ln_shape((int)cdiv(a.c, kPiece<TX>), sizeof(TX) == 2 ? 2 : 4);
  a.lg = s.lg;
  a.tiles = cdiv(a.n, s.threads >> s.lg);
  const int64_t blocks = BWD ? ln_bwd_blocks(a.tiles) : ln_blocks(a.tiles);
  if (out_blocks) *out_blocks = blocks;
  const int waves = s.lg > 6 ? 1 << (s.lg - 6) : 1;
  const size_t lds = BWD && a.partial ? (size_t)((s.threads / 64) / waves - 1) * a.c * sizeof(float) : 0;
#define M3D_LN_CASE(KK)                                                                                  \
  case KK:                                                                                               \
    return s.threads == 256 ? ln_launch_k<TX, TR, ADD, BWD, KK, 256>(a, blocks, lds, stream)              \
                            : ln_launch_k<TX, TR, ADD, BWD, KK, 1024>(a, blocks, lds, stream);
  switch (s.k) {
    M3D_LN_CASE(1)
    M3D_LN_CASE(2)
    case 3:
      if constexpr (sizeof(TX) == 4)
        return s.threads == 256 ? ln_launch_k<TX, TR, ADD, BWD, 3, 256>(a, blocks, lds, stream)
                                : ln_launch_k<TX, TR, ADD, BWD, 3, 1024>(a, blocks, lds, stream);
      break;
    case 4:
      if constexpr (sizeof(TX) == 4)
        return s.threads == 256 ? ln_launch_k<TX, TR, ADD, BWD, 4, 256>(a, blocks, lds, stream)
                                : ln_launch_k<TX, TR, ADD, BWD, 4, 1024>(a, blocks, lds, stream);
      break;
  }
#undef M3D_LN_CASE
  set_error("layer norm: no kernel for %d channels", a.c);
  return M3D_EINVAL;
}

template <bool BWD>
static int ln_dispatch(LnArgs& a, int xt, int rt, bool add, int64_t* blocks, hipStream_t s) {
  if (!add) {
    if (xt == M3D_TYPE_F32) return ln_launch<float, float, false, BWD>(a, blocks, s);
    if (xt == M3D_TYPE_BF16) return ln_launch<bf16_t, bf16_t, false, BWD>(a, blocks, s);
    return ln_launch<f16_t, f16_t, false, BWD>(a, blocks, s);
  }
  if (xt == M3D_TYPE_F32) return ln_launch<float, float, true, BWD>(a, blocks, s);
  if (xt == M3D_TYPE_BF16)
    return rt == M3D_TYPE_F32 ? ln_launch<bf16_t, float, true, BWD>(a, blocks, s)
                              : ln_launch<bf16_t, bf16_t, true, BWD>(a, blocks, s);
  return rt == M3D_TYPE_F32 ? ln_launch<f16_t, float, true, BWD>(a, blocks, s)
                            : ln_launch<f16_t, f16_t, true, BWD>(a, blocks, s);
}

static int ln_check(const char* who, int type, int stream_type, int64_t n, int c, int wtype, const void* const* ptrs,
                    const int* types, int count) {
  M3D_CHECK_ARG(type_ok(type) && type_ok(wtype), "%s: unknown element type", who);
  M3D_CHECK_ARG(stream_type == type || stream_type == M3D_TYPE_F32,
                "%s: the residual stream is of the activations' type or f32", who);
  M3D_CHECK_ARG(wtype == type || wtype == M3D_TYPE_F32, "%s: weight and bias are of the activations' type or f32", who);
  M3D_CHECK_ARG(c >= 1 && c <= kLnMaxChannels, "%s: channel count %d is not in 1..%d", who, c, kLnMaxChannels);
  M3D_CHECK_ARG(n >= 0 && n < (int64_t)1 << 32, "%s: row count %lld is not in 0..2^32-1", who, (long long)n);
  for (int i = 0; i < count; ++i)
    M3D_CHECK_ARG(((uintptr_t)ptrs[i] & (type_bytes(types[i]) - 1)) == 0, "%s: misaligned pointer", who);
  return M3D_OK;
}

static int ld_check(const char* who, int64_t n, int c, int64_t ld) {
  M3D_CHECK_ARG(ld >= c || n <= 1, "%s: row stride %lld is smaller than the %d channels", who, (long long)ld, c);
  return M3D_OK;
}

static int ln_backward(const char* who, LnArgs& a, int type, int stream_type, bool add, void* d_dweight, void* d_dbias,
                       void* d_ws, size_t ws_bytes, hipStream_t stream) {
  const bool columns = d_dweight || d_dbias;
  if (a.n == 0) {  // no rows: the column sums are zero, and there is no launch that would write them
    if (columns) {
      hipLaunchKernelGGL(ln_columns_kernel, dim3((unsigned)cdiv(2 * a.c, 32)), dim3(1024), 0, stream, nullptr, 0, a.c,
                         a.wtype, d_dweight, d_dbias);
      M3D_LAUNCH_CHECK();
    }
    return M3D_OK;
  }
  if (columns) {
    const size_t need = m3d_layer_norm_workspace_bytes(a.n, a.c, type);
    if (d_ws == nullptr || ws_bytes < need) {
      set_error("%s: workspace too small (%zu given, %zu needed)", who, ws_bytes, need);
      return M3D_ENOSPC;
    }
    M3D_CHECK_ARG(((uintptr_t)d_ws & 15) == 0, "%s: the workspace must be 16-byte aligned", who);
    a.partial = static_cast<float*>(d_ws);
  }
  int64_t blocks = 0;
  if (int rc = ln_dispatch<true>(a, type, stream_type, add, &blocks, stream)) return rc;
  if (columns) {
    hipLaunchKernelGGL(ln_columns_kernel, dim3((unsigned)cdiv(2 * a.c, 32)), dim3(1024), 0, stream, a.partial, (int)blocks,
                       a.c, a.wtype, d_dweight, d_dbias);
    M3D_LAUNCH_CHECK();
  }
  return M3D_OK;
}

}  // namespace m3d

using namespace m3d;

extern "C" size_t m3d_layer_norm_workspace_bytes(int64_t n, int c, int type) {
  if (n <= 0 || c <= 0 || c > kLnMaxChannels || !type_ok(type)) return 256;
  const LnShape s = type == M3D_TYPE_F32 ? ln_shape((int)cdiv(c, 4), 4) : ln_shape((int)cdiv(c, 8), 2);
  return align_up((size_t)ln_bwd_blocks(cdiv(n, s.threads >> s.lg)) * 2 * c * sizeof(float));
}

extern "C" int m3d_layer_norm_fwd(const void* d_x, int64_t ldx, int type, int64_t n, int c, const void* d_weight,
                                  const void* d_bias, int wtype, float eps, void* d_y, float* d_mean, float* d_rstd,
                                  void* stream) {
  const char* who = "m3d_layer_norm_fwd";
  const void* ptrs[] = {d_x, d_y, d_weight, d_bias, d_mean, d_rstd};
  const int types[] = {type, type, wtype, wtype, M3D_TYPE_F32, M3D_TYPE_F32};
  if (int rc = ln_check(who, type, type, n, c, wtype, ptrs, types, 6)) return rc;
  M3D_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", who);
  if (n == 0) return M3D_OK;
  M3D_CHECK_ARG(d_x && d_y && d_mean && d_rstd, "%s: null pointer", who);
  if (int rc = ld_check(who, n, c, ldx)) return rc;
  LnArgs a = {};
  a.in = d_x; a.ld_in = ldx; a.weight = d_weight; a.bias = d_bias; a.wtype = wtype;
  a.n = n; a.c = c; a.inv_c = 1.f / (float)c; a.eps = eps; a.y = d_y; a.mean = d_mean; a.rstd = d_rstd;
  return ln_dispatch<false>(a, type, type, false, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int m3d_layer_norm_backward(const void* d_x, int64_t ldx, const void* d_dy, int64_t lddy, int type, int64_t n,
                                       int c, const float* d_mean, const float* d_rstd, const void* d_weight, int wtype,
                                       void* d_dx, void* d_dweight, void* d_dbias, void* d_ws, size_t ws_bytes,
                                       void* stream) {
  const char* who = "m3d_layer_norm_backward";
  const void* ptrs[] = {d_x, d_dy, d_dx, d_weight, d_dweight, d_dbias, d_mean, d_rstd};
  const int types[] = {type, type, type, wtype, wtype, wtype, M3D_TYPE_F32, M3D_TYPE_F32};
  if (int rc = ln_check(who, type, type, n, c, wtype, ptrs, types, 8)) return rc;
  if (n > 0) {
    M3D_CHECK_ARG(d_x && d_dy && d_mean && d_rstd && d_dx, "%s: null pointer", who);
    if (int rc = ld_check(who, n, c, ldx)) return rc;
    if (int rc = ld_check(who, n, c, lddy)) return rc;
  }
  LnArgs a = {};
  a.in = d_x; a.ld_in = ldx; a.dy = d_dy; a.ld_dy = lddy; a.weight = d_weight; a.wtype = wtype;
  a.n = n; a.c = c; a.inv_c = 1.f / (float)c;
  a.mean = const_cast<float*>(d_mean); a.rstd = const_cast<float*>(d_rstd); a.dx = d_dx;
  return ln_backward(who, a, type, type, false, d_dweight, d_dbias, d_ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int m3d_dropout_add_layer_norm_fwd(const void* d_x, int64_t ldx, int type, const void* d_residual, int64_t ldr,
                                              int stream_type, int64_t n, int c, const void* d_weight, const void* d_bias,
                                              int wtype, float eps, double p, uint64_t seed, uint64_t offset,
                                              const int64_t* d_state, void* d_h, void* d_y, float* d_mean, float* d_rstd,
                                              void* stream) {
  const char* who = "m3d_dropout_add_layer_norm_fwd";
  const void* ptrs[] = {d_x, d_residual, d_h, d_y, d_weight, d_bias, d_mean, d_rstd};
  const int types[] = {type, stream_type, stream_type, type, wtype, wtype, M3D_TYPE_F32, M3D_TYPE_F32};
  if (int rc = ln_check(who, type, stream_type, n, c, wtype, ptrs, types, 8)) return rc;
  M3D_CHECK_ARG(eps >= 0.f, "%s: eps must not be negative", who);
  LnArgs a = {};
  if (int rc = drop_args(who, p, seed, offset, d_state, &a.drop)) return rc;
  if (n == 0) return M3D_OK;
  M3D_CHECK_ARG(d_x && d_residual && d_y && d_mean && d_rstd, "%s: null pointer", who);
  if (int rc = ld_check(who, n, c, ldx)) return rc;
  if (int rc = ld_check(who, n, c, ldr)) return rc;
  a.in = d_x; a.ld_in = ldx; a.residual = d_residual; a.ld_res = ldr; a.weight = d_weight; a.bias = d_bias;
  a.wtype = wtype; a.n = n; a.c = c; a.inv_c = 1.f / (float)c; a.eps = eps;
  a.y = d_y; a.h = d_h; a.mean = d_mean; a.rstd = d_rstd;
  return ln_dispatch<false>(a, type, stream_type, true, nullptr, static_cast<hipStream_t>(stream));
}

extern "C" int m3d_dropout_add_layer_norm_backward(const void* d_h, int64_t ldh, int stream_type, const void* d_dy,
                                                   int64_t lddy, int type, const void* d_dh, int64_t lddh, int64_t n,
                                                   int c, const float* d_mean, const float* d_rstd, const void* d_weight,
                                                   int wtype, double p, uint64_t seed, uint64_t offset,
                                                   const int64_t* d_state, void* d_dx, void* d_dresidual, void* d_dweight,
                                                   void* d_dbias, void* d_ws, size_t ws_bytes, void* stream) {
  const char* who = "m3d_dropout_add_layer_norm_backward";
  const void* ptrs[] = {d_h, d_dy, d_dh, d_dx, d_dresidual, d_weight, d_dweight, d_dbias, d_mean, d_rstd};
  const int types[] = {stream_type, type, stream_type, type, stream_type, wtype, wtype, wtype, M3D_TYPE_F32, M3D_TYPE_F32};
  if (int rc = ln_check(who, type, stream_type, n, c, wtype, ptrs, types, 10)) return rc;
  LnArgs a = {};
  if (int rc = drop_args(who, p, seed, offset, d_state, &a.drop)) return rc;
  if (n > 0) {
    M3D_CHECK_ARG(d_h && d_dy && d_mean && d_rstd && (d_dx || d_dresidual), "%s: null pointer", who);
    if (int rc = ld_check(who, n, c, ldh)) return rc;
    if (int rc = ld_check(who, n, c, lddy)) return rc;
    if (d_dh)
      if (int rc = ld_check(who, n, c, lddh)) return rc;
  }
  a.in = d_h; a.ld_in = ldh; a.dy = d_dy; a.ld_dy = lddy; a.dh = d_dh; a.ld_dh = lddh; a.weight = d_weight;
  a.wtype = wtype; a.n = n; a.c = c; a.inv_c = 1.f / (float)c;
  a.mean = const_cast<float*>(d_mean); a.rstd = const_cast<float*>(d_rstd); a.dx = d_dx; a.dres = d_dresidual;
  return ln_backward(who, a, type, stream_type, true, d_dweight, d_dbias, d_ws, ws_bytes,
                     static_cast<hipStream_t>(stream));
}
