// Layer norm over the channels of every row of [n, c] activations, forward and backward, alone and behind the residual
// add of a block:
//   alone:  y = (x - mean) * rstd * weight + bias,  mean and rstd = 1 / sqrt(var + eps) of the row
//   add:    h = residual + dropout(x) (rounded to the stream's type), y = layer norm of h as it is held
//   backward, with hat = (x - mean) * rstd and g = dy * weight:
//           dx = rstd * (g - mean(g) - hat * mean(g * hat)) [+ dh, and dropout's mask for x's own gradient]
//           dweight = sum over rows of dy * hat,  dbias = sum over rows of dy
//
// A row is held by a group of lanes in registers (K pieces of 16 bytes a lane), so that every input is read once:
// the mean, the deviations from it (their mean, which corrects it, and their squares) and the output come from the same
// registers.  Groups inside a wave add by lane permutations, wider rows take a group of several waves that add through
// LDS.  All sums are f32.
// The column sums of the backward pass stay in registers over all rows of a workgroup, are joined inside it, written as
// one partial row per workgroup and added up by a second launch in a fixed order (no atomics: run-to-run identical).
//
// Bound by HBM: 2 values moved for each forward, 3 for each backward (4 and 5 with the add), about 20 operations a value.
// Kernel times, with 2 x FETCH_SIZE + WRITE_SIZE within 2 % of those bytes: 273080 x 96 f32 35.9 us forward (5.8 TB/s),
// 53.9 backward (5.8); 75401 x 768 bf16 39.8 and 59.0 (5.8, 5.9); 16384 x 4096 bf16 with dropout and add 102.8 (5.2) and
// 123.9 (5.4); the join of the columns 4.7.  A copy of 1 GB runs at 5.2.  Where a workgroup gets few rows the partial rows
// weigh more: 3493 x 1001 f16 backward moves 32 % above its 21 MB in the first launch, and 6 MB again in the join.
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
template <int THREADS>
struct RowSum {
  float (*red)[THREADS / 64][2];
  int turn = 0;
  template <int NQ>
  __device__ __forceinline__ void operator()(float (&v)[NQ], int lg) {
    static_assert(NQ <= 2, "a slot holds two sums");
    const int g = 1 << lg;
    group_sum(v, g < 64 ? g : 64);
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

// A lane's pieces k = 0 .. K - 1 are lane + k * g: the same for every row, and whole but for the last.  Addresses are a
// uniform 64-bit base per tile (scalar registers) and a 32-bit byte offset per lane.
template <int K, int V, bool RAGGED>
struct Lane {
  int g, lane, slot, c;
  Place last;
  __device__ __forceinline__ Lane(const LnArgs& a, int lg) : g(1 << lg), c(a.c) {
    lane = threadIdx.x & (g - 1);
    slot = threadIdx.x >> lg;
    last = place_of<V>(lane + (K - 1) * g, c);
  }
  __device__ __forceinline__ Place at(int k) const {
    return k == K - 1 ? last : Place{(lane + k * g) * V, 0, V};
  }
  // loads of piece k: `base` = the tile's first row, `row` = this lane's row in it
  template <typename T>
  __device__ __forceinline__ void load(Piece<T, V>& q, int k, const T* base, int64_t ld, int row) const {
    const Place p = at(k);
    const uint32_t off = (uint32_t)row * (uint32_t)ld + (uint32_t)p.col;
    if constexpr (!RAGGED) q.load_stream(base + off);
    else if (p.count < V) q.load_some(base + off, 0, p.count);
    else q.load(base + off);
  }
  template <typename T>
  __device__ __forceinline__ void store(const Piece<T, V>& q, int k, T* base, int row) const {
    const Place p = at(k);
    const uint32_t off = (uint32_t)row * (uint32_t)c + (uint32_t)p.col;
    if (p.skip == 0 && p.count == V) q.store(base + off);
    else if (RAGGED && p.skip < V) q.store_some(base + off, p.skip, p.count);
  }
  // is position i of piece k this lane's own?
  __device__ __forceinline__ bool own(int k, int i) const {
    if (k < K - 1) return true;
    return RAGGED ? i >= last.skip && i < last.count : last.skip == 0;
  }
  __device__ __forceinline__ void drop(float* v, int k, uint32_t row, const DropKey& key, const DropArgs& d) const {
    const Place p = at(k);
    if (RAGGED && p.skip > 0) {
      if (p.skip < V) drop_unaligned<V>(v, p.col, row, key, d.last, d.scale);
    } else {
      m3d::drop<V>(v, p.col, row, key, d.last, d.scale);
    }
  }
};

// a * b as rounded: not contracted into the additions that use it, each of which would see another value
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// Alone, the norm is held to the 128 registers at which the chip holds the workgroups that ln_blocks starts (65 bf16
// channels 4.0 TB/s, with the 129 that it would take 3.2).  With the add some rows need more and would spill.
template <typename TX, typename TR, int K, bool ADD, bool RAGGED, int THREADS>
__global__ __launch_bounds__(THREADS, ADD ? 1 : 4) void ln_fwd_kernel(LnArgs a) {
  constexpr int V = kPiece<TX>;
  __shared__ float red[2][THREADS / 64][2];
  RowSum<THREADS> row_sum{red};
  const Lane<K, V, RAGGED> at(a, a.lg);
  const int rows = THREADS >> a.lg;
  DropKey key = {};
  if (ADD && a.drop.on) key = drop_key(a.drop);
  float w[K][V], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_params<V>(a.weight, a.wtype, at.at(k), 1.f, w[k]);
    load_params<V>(a.bias, a.wtype, at.at(k), 0.f, b[k]);
  }
  // The next tile's pieces are requested before this tile is reduced and written.
  Piece<TX, V> x[K];
  Piece<TR, V> r[ADD ? K : 1];
  auto fetch = [&](int64_t tile) {
    const int64_t first = tile * rows;
    const int row = a.n - first < rows && at.slot >= (int)(a.n - first) ? (int)(a.n - first) - 1 : at.slot;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at.load(x[k], k, static_cast<const TX*>(a.in) + first * a.ld_in, a.ld_in, row);
      if constexpr (ADD) at.load(r[k], k, static_cast<const TR*>(a.residual) + first * a.ld_res, a.ld_res, row);
    }
  };
  int64_t tile = blockIdx.x;
  if (tile < a.tiles) fetch(tile);
  for (; tile < a.tiles; tile += gridDim.x) {
    const int64_t first = tile * rows;
    const bool live = at.slot < a.n - first;  // a row behind the last one is computed as a copy of it and not stored
    float v[K][V], s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = x[k].get(i);
      if constexpr (ADD) {
        if (a.drop.on) at.drop(v[k], k, (uint32_t)(first + at.slot), key, a.drop);
        Piece<TR, V> h;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h.set(i, r[k].get(i) + v[k][i]);
          v[k][i] = h.get(i);
        }
        if (a.h && live) at.store(h, k, static_cast<TR*>(a.h) + first * a.c, at.slot);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += at.own(k, i) ? v[k][i] : 0.f;
    }
    if (tile + gridDim.x < a.tiles) fetch(tile + gridDim.x);
    row_sum(s, a.lg);
    // The mean is off by the rounding of its sum, a few steps of the row's magnitude, which may be as large as sqrt(eps) or
    // as the deviations themselves (96 equal values between 1000 and 2000 gave |y| up to 0.12).  The deviations are exact
    // there, so their own mean is added back to it and taken out of them and, squared, of the variance.  The second sum
    // costs nothing where the memory binds (forward and backward of 273080 x 96 f32 101 us, 8192 x 8192 bf16 forward 44.4
    // us, with and without); rows of sixteen waves wait for it (16384 bf16 channels 4.8 TB/s, without 5.2; f32 6.2, 6.3).
    const float about = rounded_product(s[0], a.inv_c);
    float dev[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[k][i] = at.own(k, i) ? v[k][i] - about : 0.f;
        dev[0] += v[k][i];
        dev[1] += v[k][i] * v[k][i];
      }
    row_sum(dev, a.lg);
    const float shift = rounded_product(dev[0], a.inv_c), square = dev[1] * a.inv_c;
    const float mean = about + shift;
    float var = square - shift * shift;
    if (var < 0.f) var = 0.f;
    if (square == __builtin_inff()) var = square;  // squares that overflow leave y = bias, whatever the shift's did
    const float rstd = 1.f / __builtin_sqrtf(var + a.eps), scaled = shift * rstd;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      Piece<TX, V> y;
#pragma unroll
      for (int i = 0; i < V; ++i) y.set(i, __builtin_fmaf(__builtin_fmaf(v[k][i], rstd, -scaled), w[k][i], b[k][i]));
      if (live) at.store(y, k, static_cast<TX*>(a.y) + first * a.c, at.slot);
    }
    if (at.lane == 0 && live) {
      a.mean[first + at.slot] = mean;
      a.rstd[first + at.slot] = rstd;
    }
  }
}

// Hides from the compiler that the piece still holds what it held, so that nothing formed from it is kept in registers.
template <typename T, int V>
__device__ __forceinline__ void keep_packed(Piece<T, V>& q) {
  typedef unsigned words __attribute__((ext_vector_type(V * sizeof(T) / 4)));
  words w = __builtin_bit_cast(words, q.v);
#pragma unroll
  for (int i = 0; i < (int)(V * sizeof(T) / 4); ++i) {
    unsigned one = w[i];
    asm volatile("" : "+v"(one));
    w[i] = one;
  }
  q.v = __builtin_bit_cast(typename Piece<T, V>::vec, w);
}

template <typename TX, typename TR, int K, bool ADD, bool RAGGED, int THREADS>
__global__ __launch_bounds__(THREADS) void ln_bwd_kernel(LnArgs a) {
  constexpr int V = kPiece<TX>;
  __shared__ float red[2][THREADS / 64][2];
  RowSum<THREADS> row_sum{red};
  const Lane<K, V, RAGGED> at(a, a.lg);
  const int rows = THREADS >> a.lg, c = a.c;
  DropKey key = {};
  if (ADD && a.drop.on) key = drop_key(a.drop);
  // The weight is read from LDS for every row ([V / 4][pieces][4], conflict-free): it would take K * V registers, which
  // the pieces in flight need.
  extern __shared__ float lds[];  // [max(slots / 2, 1)][channels up to whole pieces]: the weight, later the joins
  const int pieces = at.g * K;
  for (int q = threadIdx.x; q < pieces; q += THREADS) {
    float v[V];
    load_params<V>(a.weight, a.wtype, place_of<V>(q, c), 1.f, v);
#pragma unroll
    for (int i = 0; i < V; ++i) lds[((i >> 2) * pieces + q) * 4 + (i & 3)] = v[i];
  }
  __syncthreads();
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  Piece<TR, V> x[K], dh[ADD ? K : 1];
  Piece<TX, V> dy[K];
  float mean, rstd;
  auto fetch = [&](int64_t tile) {
    const int64_t first = tile * rows;
    const int row = a.n - first < rows && at.slot >= (int)(a.n - first) ? (int)(a.n - first) - 1 : at.slot;
    mean = a.mean[first + row];
    rstd = a.rstd[first + row];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at.load(x[k], k, static_cast<const TR*>(a.in) + first * a.ld_in, a.ld_in, row);
      at.load(dy[k], k, static_cast<const TX*>(a.dy) + first * a.ld_dy, a.ld_dy, row);
    }
  };
  // A workgroup of 1024 has 128 registers a lane: there the pieces stay packed and what the second pass needs is formed
  // again from them, with no tile in flight (4096 x 16384 bf16 with the add: 3.3 TB/s; kept as floats and a tile ahead the
  // spilled registers leave 2.4).
  constexpr bool kPacked = THREADS == 1024;
  int64_t tile = blockIdx.x;
  if (!kPacked && tile < a.tiles) fetch(tile);
  for (; tile < a.tiles; tile += gridDim.x) {
    const int64_t first = tile * rows;
    const bool live = at.slot < a.n - first;
    if constexpr (kPacked) fetch(tile);
    if constexpr (ADD)
      if (a.dh) {
        const int row = live ? at.slot : (int)(a.n - first) - 1;
#pragma unroll
        for (int k = 0; k < K; ++k) at.load(dh[k], k, static_cast<const TR*>(a.dh) + first * a.ld_dh, a.ld_dh, row);
      }
    float hat[K][V], gw[K][V], s[2] = {0.f, 0.f};
    const float scale = rstd;
    // position i of piece k: its normalised input and the gradient behind the weight.  Neither a row behind the last one
    // nor another lane's channel adds to a sum.
    auto form = [&](int k, int i, float& h, float& d) {
      h = (x[k].get(i) - mean) * rstd;
      d = live && at.own(k, i) ? dy[k].get(i) : 0.f;
      return d * lds[((i >> 2) * pieces + at.lane + k * at.g) * 4 + (i & 3)];
    };
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float d;
        gw[k][i] = form(k, i, hat[k][i], d);
        dw[k][i] += d * hat[k][i];
        db[k][i] += d;
        s[0] += gw[k][i];
        s[1] += gw[k][i] * hat[k][i];
      }
    if (!kPacked && tile + gridDim.x < a.tiles) fetch(tile + gridDim.x);
    row_sum(s, a.lg);
    const float m0 = s[0] * a.inv_c, m1 = s[1] * a.inv_c;
    if constexpr (kPacked) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        keep_packed(x[k]);
        keep_packed(dy[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (kPacked) {
          float d;
          gw[k][i] = form(k, i, hat[k][i], d);
        }
        v[i] = (gw[k][i] - m0 - hat[k][i] * m1) * scale;
        if constexpr (ADD)
          if (a.dh) v[i] += dh[k].get(i);
      }
      if constexpr (ADD) {
        Piece<TR, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.set(i, v[i]);
        if (a.dres && live) at.store(out, k, static_cast<TR*>(a.dres) + first * c, at.slot);
        if (a.drop.on) at.drop(v, k, (uint32_t)(first + at.slot), key, a.drop);
      }
      Piece<TX, V> out;
#pragma unroll
      for (int i = 0; i < V; ++i) out.set(i, v[i]);
      if (a.dx && live) at.store(out, k, static_cast<TX*>(a.dx) + first * c, at.slot);
    }
  }
  if (a.partial == nullptr) return;
  // The groups of a workgroup that hold the same channels are joined: lanes of a wave by shuffles, then the upper half of
  // the waves' sums through LDS onto the lower half until one is left (a group of several waves owns its channels
  // alone within its slot).
  const int g = at.g;
  for (int o = g; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        dw[k][i] += __shfl_xor(dw[k][i], o);
        db[k][i] += __shfl_xor(db[k][i], o);
      }
  const int waves = g > 64 ? g >> 6 : 1;
  const int me = (threadIdx.x >> 6) / waves;
  const bool mine = (int)(threadIdx.x & 63) < g;
  const int lane = at.lane;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float(&sum)[K][V] = q ? db : dw;
    for (int half = (THREADS / 64) / waves / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (me >= half && me < 2 * half && mine)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) lds[((me - half) * V + i) * pieces + lane + k * g] = sum[k][i];
      __syncthreads();
      if (me < half && mine)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) sum[k][i] += lds[(me * V + i) * pieces + lane + k * g];
    }
    if (me == 0 && mine)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        Piece<float, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.set(i, sum[k][i]);
        at.store(o, k, a.partial + ((int64_t)blockIdx.x * 2 + q) * c, 0);
      }
  }
}

// dweight and dbias from the partial rows, in f64 and in a fixed order: a workgroup owns 32 columns of the 2 * c, each of
// its 32 row groups adds every 32nd partial row, eight loads in flight, and the group sums are joined by halves.
__global__ __launch_bounds__(1024) void ln_columns_kernel(const float* __restrict__ partial, int blocks, int c, int wtype,
                                                          void* dweight, void* dbias) {
  constexpr int kInFlight = 8;
  __shared__ double red[32][33];
  const int e = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + e;
  const float* p = partial + (col < 2 * c ? col : 0);
  double s = 0.0;
  int r = grp;
  for (; r + 32 * (kInFlight - 1) < blocks; r += 32 * kInFlight) {
    float v[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) v[i] = p[(int64_t)(r + 32 * i) * 2 * c];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) s += (double)v[i];
  }
  for (; r < blocks; r += 32) s += (double)p[(int64_t)r * 2 * c];
  red[grp][e] = s;
  for (int half = 16; half > 0; half >>= 1) {
    __syncthreads();
    if (grp < half) red[grp][e] += red[grp + half][e];
  }
  if (grp == 0 && col < 2 * c) {
    const float t = (float)red[0][e];
    void* to = col < c ? dweight : dbias;
    const int at = col < c ? col : col - c;
    if (to == nullptr) return;
    if (wtype == M3D_TYPE_F32) static_cast<float*>(to)[at] = t;
    else if (wtype == M3D_TYPE_BF16) static_cast<bf16_t*>(to)[at] = (bf16_t)t;
    else static_cast<f16_t*>(to)[at] = (f16_t)t;
  }
}

// ---------------------------------------------------------------- launch shapes
constexpr int kLnMaxChannels = 16384;
constexpr int kLnMaxStride = 1 << 20;  // elements: a tile's rows (256 at most) stay within 32-bit offsets

struct LnShape {
  int lg, k, threads;
};

// Lanes and pieces a lane for a row of `pieces` 16-byte pieces: the (lanes, K) that leave the fewest places empty, the
// larger K where two leave the same.  Rows of whole pieces take 8 lanes or more, so that a load covers whole lines (40
// bf16 channels forward: 4.2 TB/s, on 2 lanes 3.7); other rows are bound by their lanes' work and may take 2 (65 bf16
// channels forward: 4.0 TB/s, on 8 lanes 3.1).
static LnShape ln_shape(int c, int type) {
  const int v = type == M3D_TYPE_F32 ? 4 : 8, pieces = (int)cdiv(c, v), g_min = c % v == 0 ? 8 : 2;
  LnShape best = {0, 0, 0};
  int waste = 0;
  for (int lg = 0; lg <= 10; ++lg) {
    const int g = 1 << lg, k = (int)cdiv(pieces, g);
    if (k > (lg < 10 ? 3 : 4) || (g < g_min && g < pieces)) continue;
    if (best.k == 0 || g * k < waste) {
      best = {lg, k, lg > 9 ? 1024 : lg > 8 ? 512 : 256};
      waste = g * k;
    }
  }
  return best;
}

// Workgroups: every one walks over its tiles with the next tile's pieces in flight, so that a few waves keep the memory
// busy, and each costs a load of weight and bias, or a partial row of column sums.
//   forward:   as many as the chip holds at 1024 threads a CU (273080 x 96 f32: 37.4 us; with half as many on rows of
//              8192 bf16 channels 56 against 47.6 us, with four times as many 59)
//   backward:  512 threads a CU, or 768 where a lane has 64 bytes in flight or fewer (500000 x 32 f32: 39 against 44 us;
//              75401 x 768 bf16, 96 bytes: 71 with 512 against 83 with 768, which no longer fit the registers at once).
//              Rows of a group of 256 lanes take workgroups of 512, two rows at a time: half the partial rows.  Rows
//              of 1024 lanes are a workgroup each, 1024 threads a CU.
constexpr int kLnCus = 256;
static LnShape ln_bwd_shape(int c, int type) {
  LnShape s = ln_shape(c, type);
  if (s.lg == 8) s.threads = 512;
  return s;
}
static int64_t ln_blocks(int64_t tiles, int threads) {
  const int64_t most = kLnCus * 1024 / threads;
  return tiles < most ? tiles : most;
}
static int64_t ln_bwd_blocks(int64_t tiles, const LnShape& s, int bytes_in_flight) {
  const int64_t most = s.threads > 256 ? kLnCus : bytes_in_flight <= 64 ? 3 * kLnCus : 2 * kLnCus;
  return tiles < most ? tiles : most;
}

template <typename TX, typename TR, bool ADD, bool BWD, int K, bool RAGGED, int THREADS>
static int ln_launch_t(LnArgs& a, int64_t blocks, size_t lds, hipStream_t stream) {
  const dim3 grid((unsigned)blocks), block(THREADS);
  if constexpr (BWD) {
    static LdsGrant grant;
    auto kernel = ln_bwd_kernel<TX, TR, K, ADD, RAGGED, THREADS>;
    if (lds > 60 * 1024)  // below the 64 KB that every kernel may have
      if (int rc = grant.ensure(reinterpret_cast<const void*>(kernel), lds)) return rc;
    hipLaunchKernelGGL(kernel, grid, block, lds, stream, a);
  } else {
    hipLaunchKernelGGL((ln_fwd_kernel<TX, TR, K, ADD, RAGGED, THREADS>), grid, block, 0, stream, a);
  }
  M3D_LAUNCH_CHECK();
  return M3D_OK;
}

template <typename TX, typename TR, bool ADD, bool BWD, int K, bool RAGGED>
static int ln_launch_k(LnArgs& a, const LnShape& s, int64_t blocks, size_t lds, hipStream_t stream) {
  // what ln_shape reaches: one piece a lane only in rows of 8 pieces or fewer, four only in the widest f32 rows
  if constexpr (K <= 3)
    if (s.threads == 256) return ln_launch_t<TX, TR, ADD, BWD, K, RAGGED, 256>(a, blocks, lds, stream);
  if constexpr (K == 2 || K == 3)
    if (s.threads == 512) return ln_launch_t<TX, TR, ADD, BWD, K, RAGGED, 512>(a, blocks, lds, stream);
  if constexpr (K == 2 || (K > 2 && sizeof(TX) == 4))
    if (s.threads == 1024) return ln_launch_t<TX, TR, ADD, BWD, K, RAGGED, 1024>(a, blocks, lds, stream);
  set_error("layer norm: no kernel for %d channels", a.c);
  return M3D_EINVAL;
}

template <typename TX, typename TR, bool ADD, bool BWD>
static int ln_launch(LnArgs& a, int64_t* out_blocks, hipStream_t stream) {
  const LnShape s = BWD ? ln_bwd_shape(a.c, TypeCode<TX>::value) : ln_shape(a.c, TypeCode<TX>::value);
  a.lg = s.lg;
  a.tiles = cdiv(a.n, s.threads >> s.lg);
  const int in_flight = s.k * kPiece<TX> * (int)(sizeof(TX) + sizeof(TR) * (ADD ? 2 : 1));
  const int64_t blocks = BWD ? ln_bwd_blocks(a.tiles, s, in_flight) : ln_blocks(a.tiles, s.threads);
  if (out_blocks) *out_blocks = blocks;
  const int slots = (s.threads / 64) / (s.lg > 6 ? 1 << (s.lg - 6) : 1);
  const size_t lds = BWD ? (size_t)(slots > 2 && a.partial ? slots / 2 : 1) * (s.k << s.lg) * kPiece<TX> * sizeof(float) : 0;
  const bool ragged = a.c % kPiece<TX> != 0;
#define M3D_LN_CASE(KK)                                                                        \
  case KK:                                                                                     \
    return ragged ? ln_launch_k<TX, TR, ADD, BWD, KK, true>(a, s, blocks, lds, stream)          \
                  : ln_launch_k<TX, TR, ADD, BWD, KK, false>(a, s, blocks, lds, stream);
  switch (s.k) {
    M3D_LN_CASE(1)
    M3D_LN_CASE(2)
    M3D_LN_CASE(3)
    M3D_LN_CASE(4)
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
  M3D_CHECK_ARG(n <= 1 || (ld >= c && ld <= kLnMaxStride),
                "%s: row stride %lld is not between the %d channels and %d", who, (long long)ld, c, kLnMaxStride);
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
  const LnShape s = ln_bwd_shape(c, type);
  return align_up((size_t)ln_bwd_blocks(cdiv(n, s.threads >> s.lg), s, 0) * 2 * c * sizeof(float));  // the most of all
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
