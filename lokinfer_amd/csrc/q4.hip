// Products with 4-bit weights (lk.ops.q4_gpu; no counterpart in the reference, whose weights are f16 or f32).
//
//   y[m, n] = sum_k x[m, k] s[k / G, n] (c[k, n] - 8),  x f16, codes c and scales s as in q4.h, G = 32, 64 or 128
//
//   lk_hip_w4_quantize   w f16[K, N] (or [N, K]) -> codes and scales in the layout below
//   lk_hip_w4_pack       given codes u8[K, N] and scales f16[ceil(K / G), N] -> the same layout
//   lk_hip_w4_unpack     -> f16[K, N], exact
//   lk_hip_w4_gemm       x @ W, + bias, + residual, SwiGLU of two weights, f32 logits; RMSNorm in front of one row
//
// Layout: tiles of 16 columns x 128 k, q [ceil(N / 16), ceil(K / 128), 64, 4] words: word i of lane l holds the codes of column
// l % 16, k = 32 i + 8 (l / 16) + 0 .. 7 of the tile, so a wave's 16-byte load is one contiguous KiB and its word i is the B
// operand of a 16x16x32 MFMA (two tiles' words are those of 32x32x16 ones). Scales f16 [ceil(N / 16), ceil(K / 128), 16, 128 / G].
// Columns and k past the weight's hold zeros (code 8, scale 0).
#include <algorithm>

#include "common.h"
#include "lokinfer_hip.h"
#include "q4.h"

namespace lkd {

struct W4Layout {
  int64_t n, k, kb;  // logical sizes; kb = ceil(K / 128)
  int group;
};

// One thread per (column of a tile, group), from w f16[K, N] (neighbouring threads on neighbouring columns) or NT f16[N, K]
// (on neighbouring groups). The group's values stay in registers between the search for its scale and the codes. Runs once per
// weight: 2048 x 12288 34 us (1.9 TB/s), NT 151936 x 2048 0.26 ms (3.0 TB/s).
template <bool NT, int G>
__global__ __launch_bounds__(256) void w4QuantizeKernel(const h16* __restrict__ w, unsigned* __restrict__ q,
                                                        h16* __restrict__ s, W4Layout p, bool wide) {
  constexpr int PER = 128 / G;
  const int64_t cols = (p.n + 15) / 16 * 16, groups = p.kb * PER, total = cols * groups;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t major = id / (NT ? groups : cols), minor = id - major * (NT ? groups : cols);
    const int64_t n = NT ? major : minor, gi = NT ? minor : major, kb = gi / PER, k0 = gi * G;
    const int gb = static_cast<int>(gi - kb * PER);
    const int live = n < p.n ? static_cast<int>(max<int64_t>(0, min<int64_t>(G, p.k - k0))) : 0;
    half8 v[G / 8];
#pragma unroll
    for (int o = 0; o < G / 8; ++o) v[o] = half8{};
    const auto at = [&](int j) { return NT ? w[n * p.k + k0 + j] : w[(k0 + j) * p.n + n]; };
#pragma unroll
    for (int o = 0; o < G / 8; ++o) {
      if (live == G) {
        if (NT && wide) {
          v[o] = ld8(w + n * p.k + k0 + 8 * o);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[o][e] = at(8 * o + e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * o + e < live) v[o][e] = at(8 * o + e);
      }
    }
    float hi = 0.0f, lo = 0.0f;
    bool bad = false;
#pragma unroll
    for (int o = 0; o < G / 8; ++o)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = static_cast<float>(v[o][e]);
        hi = fmaxf(hi, x);
        lo = fminf(lo, x);
        bad = bad || !(fabsf(x) < INFINITY);
      }
    const float sc = bad ? __builtin_nanf("") : q4Scale(hi, lo);
    const int64_t tile = (n >> 4) * p.kb + kb;
    s[(tile * 16 + (n & 15)) * PER + gb] = static_cast<h16>(sc);
#pragma unroll
    for (int o = 0; o < G / 8; ++o) {
      unsigned word = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) word |= q4Code(static_cast<float>(v[o][e]), sc) << q4Shift(e);  // past K: 0, code 8
      const int in = gb * G + 8 * o;  // k within the tile
      q[(tile * 64 + (n & 15) + 16 * ((in >> 3) & 3)) * 4 + (in >> 5)] = word;
    }
  }
}

// Given codes and scales: one thread per (column, 8 of each 32 k of a tile), grid columns / 64, k blocks. What is no code or no
// scale sets a flag: 1 a code over 15, 2 a scale that is negative, over 8128 or not a number, or has more than 8 bits. Runs
// once per weight: 2048 x 151936 172 us (2.8 TB/s).
__global__ __launch_bounds__(256) void w4PackKernel(const uint8_t* __restrict__ codes, const h16* __restrict__ scales,
                                                    uint4* __restrict__ q, h16* __restrict__ s, int* __restrict__ flag,
                                                    W4Layout p) {
  const int per = 128 / p.group, kq = threadIdx.x >> 6;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 64 + (threadIdx.x & 63), tiles = (p.n + 15) / 16;
  if (n >= tiles * 16) return;
  for (int64_t kb = blockIdx.y; kb < p.kb; kb += gridDim.y) {
    unsigned c[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t k = kb * 128 + 32 * i + 8 * kq + j;
        c[i][j] = n < p.n && k < p.k ? codes[k * p.n + n] : 8u;
      }
    unsigned word[4] = {0u, 0u, 0u, 0u}, all = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        word[i] |= (c[i][j] & 15u) << q4Shift(j);
        all |= c[i][j];
      }
    if (all > 15u) atomicOr(flag, 1);
    const int64_t tile = (n >> 4) * p.kb + kb;
    q[tile * 64 + (n & 15) + 16 * kq] = make_uint4(word[0], word[1], word[2], word[3]);
    if (kq < per) {
      const int64_t g = kb * per + kq;
      const h16 sc = n < p.n && g * p.group < p.k ? scales[g * p.n + n] : static_cast<h16>(0.0f);
      const unsigned bits = __builtin_bit_cast(unsigned short, sc), sub = bits & 0x3FFu;
      // normal: the last 3 of 11 bits; subnormal: an odd part under 256
      const bool fine = bits <= 0x6FF0u && (bits >= 0x400u ? (bits & 7u) == 0u : sub == 0u || (sub >> (__ffs(sub) - 1)) < 256u);
      if (!fine) atomicOr(flag, 2);
      s[(tile * 16 + (n & 15)) * per + kq] = sc;
    }
  }
}

// one thread per (8 k, column): out f16[K, N]; 2048 x 12288 21 us (3.1 TB/s)
__global__ __launch_bounds__(256) void w4UnpackKernel(const unsigned* __restrict__ q, const h16* __restrict__ s,
                                                      h16* __restrict__ out, W4Layout p) {
  const Q4Masks masks;
  const int per = 128 / p.group;
  const int64_t total = (p.k + 7) / 8 * p.n;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t k8 = id / p.n, n = id - k8 * p.n, k = 8 * k8, tile = (n >> 4) * p.kb + k / 128;
    const int in = static_cast<int>(k & 127);
    const h16 sc = s[(tile * 16 + (n & 15)) * per + in / p.group];
    const half8 v = q4Ints(q[(tile * 64 + (n & 15) + 16 * ((in >> 3) & 3)) * 4 + (in >> 5)], masks);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < p.k) out[(k + j) * p.n + n] = v[j] * sc;
  }
}

struct W4Params {
  const h16* x;       // [M, K]
  const h16* gamma;   // RMSNorm gain [K] (M = 1) or null
  const uint4* q[2];  // gate, up for SwiGLU
  const h16* s[2];
  const h16* bias;  // [N] or null
  const h16* res;   // [M, N] or null
  void* out;        // f16 (or f32) [M, N]
  int64_t m, n, k, kb;
  float eps;
};

// ---- up to 16 rows: 16x16x32 MFMAs, x as A (its row j is the operand's row 4 (j % 4) + j / 4, so that its sums are
// accumulator j / 4 of lanes 16 (j % 4) ..: few rows need only RU = ceil(rows / 4) of the 4 accumulators), 16 columns of the
// weight as B. A group's products are summed on its integers and scaled once, in f32. The weights are read once and are all the
// traffic that counts: bound by HBM where there are many, by the latency of a few dependent loads where there are few.
template <int G, int W>
struct W4Block {  // a tile's k block, as loaded
  static constexpr int PER = 128 / G;
  uint4 q[W];
  h16 s[W][PER];
  __device__ __forceinline__ void load(const W4Params& p, int64_t tile, int64_t kb, int lane) {
    const int64_t at = tile * p.kb + kb;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.q[w] + at * 64 + lane));  // read once
      q[w] = make_uint4(v[0], v[1], v[2], v[3]);
      const h16* sp = p.s[w] + (at * 16 + (lane & 15)) * PER;
#pragma unroll
      for (int g = 0; g < PER; ++g) s[w][g] = sp[g];
    }
  }
  // acc += x (the block's 4 operands) times the block
  template <int RU>
  __device__ __forceinline__ void multiply(const half8 (&x)[4], float (&acc)[W][RU], const Q4Masks& masks) const {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned word[4] = {q[w].x, q[w].y, q[w].z, q[w].w};
#pragma unroll
      for (int g = 0; g < PER; ++g) {
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = g * G / 32; i < (g + 1) * G / 32; ++i)
          d = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], q4Ints(word[i], masks), d, 0, 0, 0);
        const float f = static_cast<float>(s[w][g]);
#pragma unroll
        for (int r = 0; r < RU; ++r) acc[w][r] = fmaf(f, d[r], acc[w][r]);
      }
    }
  }
};

template <bool F32, int W>
__device__ __forceinline__ void w4Put(const W4Params& p, int64_t row, int64_t col, const float (&y)[W]) {
  if (row >= p.m || col >= p.n) return;
  if constexpr (F32) {
    static_cast<float*>(p.out)[row * p.n + col] = y[0];
  } else {
    float v = y[0];
    if constexpr (W == 2) v = siluMul(y[0], y[W - 1]);
    if (p.bias) v += static_cast<float>(p.bias[col]);
    if (p.res) v = static_cast<float>(p.res[row * p.n + col]) + v;
    static_cast<h16*>(p.out)[row * p.n + col] = toH16(v);
  }
}

// Few tiles: the WAVES waves of a workgroup share one tile's k blocks (wave w takes w, w + WAVES, ..., U at a time, all loads
// first) and their sums meet in LDS. 1 x 2048 x 4096 4.1 us (4.5 MB), 4 x 2048 x 6144 of two weights 6.8 us (14 MB, 2.1 TB/s): a
// launch that does next to nothing takes 2.5.
template <int RU, int G, int W, bool F32, bool RMS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void w4SplitKernel(W4Params p) {
  const Q4Masks masks;
  __shared__ float red[WAVES][W][RU][64];
  constexpr int U = W == 2 ? 2 : 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, kq = lane >> 4;
  const int64_t tile = blockIdx.x, row = 4 * (a & 3) + (a >> 2);
  float acc[W][RU];
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int r = 0; r < RU; ++r) acc[w][r] = 0.0f;
  // With a norm in front (one row): the row, the gains and the weights are all loaded before the first is waited for; a lane
  // normalizes one 16-byte piece of the wave's U blocks and the wave's LDS hands them round. Rows 1 .. of the operand repeat
  // row 0: their sums are not stored.
  constexpr int AHEAD = RMS ? 4 : 0;  // the lane's first pieces of the sum of squares, which has rowSumSq's order
  __shared__ __attribute__((aligned(16))) h16 normed[RMS ? WAVES : 1][U * 128];
  half8 sq[AHEAD + 1];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    sq[j] = half8{};
    if (lane + 64 * j < p.k / 8) sq[j] = ld8(p.x + 8 * (lane + 64 * j));
  }
  float rf = 1.0f;
  for (int64_t k0 = wave; k0 < p.kb; k0 += U * WAVES) {
    W4Block<G, W> blk[U];
    half8 x[U][4], piece{}, gain{};
    if constexpr (RMS) {
      const int64_t k = (k0 + (lane >> 4) * WAVES) * 128 + 8 * (lane & 15);
      if (lane < 16 * U && k < p.k) {
        piece = ld8(p.x + k);
        gain = ld8(p.gamma + k);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) blk[u].load(p, tile, min<int64_t>(k0 + u * WAVES, p.kb - 1), lane);
    if constexpr (RMS) {
      if (k0 == wave) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(static_cast<float>(sq[j][e]), static_cast<float>(sq[j][e]), sum);
        for (int64_t c = lane + 64 * AHEAD; c < p.k / 8; c += 64) {
          const half8 v = ld8(p.x + 8 * c);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum = fmaf(static_cast<float>(v[e]), static_cast<float>(v[e]), sum);
        }
        rf = rmsFactor(waveSum(sum), p.k, p.eps);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) piece[e] = rmsElem(piece[e], gain[e], rf);
      __builtin_amdgcn_wave_barrier();
      if (lane < 16 * U) st8(&normed[wave][8 * lane], piece);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[u][i] = ld8(&normed[wave][128 * u + 32 * i + 8 * kq]);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t k = (k0 + u * WAVES) * 128 + 32 * i + 8 * kq;
          x[u][i] = half8{};
          if (row < p.m && k < p.k) x[u][i] = ld8(p.x + row * p.k + k);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + u * WAVES < p.kb) blk[u].multiply(x[u], acc, masks);
  }
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int r = 0; r < RU; ++r) red[wave][w][r][lane] = acc[w][r];
  __syncthreads();
  for (int o = threadIdx.x; o < RU * 64; o += 64 * WAVES) {
    const int l = o & 63, r = o >> 6;
    float y[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      y[w] = 0.0f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) y[w] += red[v][w][r][l];
    }
    w4Put<F32, W>(p, 4 * r + (l >> 4), tile * 16 + (l & 15), y);
  }
}

// Many tiles: x (normalized with RMS) goes to LDS once per workgroup, then each wave streams tiles of its own, U k blocks
// ahead, over the tiles' ends. 1 x 2048 x 151936 30.7 us: 166 MB at 5.4 TB/s, above what a large copy reaches (4.7); 4 rows 33,
// 16 rows 53, with two workgroups a CU beside their 67 KB of x.
constexpr int kStreamPad = 32;  // halves between x's rows in LDS
template <int RU, int G, int W, bool F32, bool RMS>
__global__ __launch_bounds__(256) void w4StreamKernel(W4Params p) {
  const Q4Masks masks;
  extern __shared__ __attribute__((aligned(16))) h16 xs[];  // [M][kb 128 + kStreamPad]
  constexpr int U = 4 / W;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, kq = lane >> 4;
  const int64_t ld = p.kb * 128 + kStreamPad;
  float rf = 1.0f;
  if constexpr (RMS) rf = rmsFactor(rowSumSq(p.x, p.k, lane), p.k, p.eps);
  for (int64_t i = threadIdx.x; i < p.m * p.kb * 16; i += 256) {
    const int64_t row = i / (p.kb * 16), k = (i - row * p.kb * 16) * 8;
    half8 v = {};
    if (k < p.k) {
      v = ld8(p.x + row * p.k + k);
      if constexpr (RMS) {
        const half8 gv = ld8(p.gamma + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = rmsElem(v[e], gv[e], rf);
      }
    }
    st8(xs + row * ld + k, v);
  }
  __syncthreads();
  const int64_t tiles = (p.n + 15) / 16, step = static_cast<int64_t>(gridDim.x) * 4;
  const int64_t batches = (p.kb + U - 1) / U;
  // rows past M read row 0: their sums are not used
  const int64_t rowOf = 4 * (a & 3) + (a >> 2);
  const h16* xr = xs + (rowOf < p.m ? rowOf : 0) * ld + 8 * kq;
  int64_t tile = blockIdx.x * 4 + wave;
  if (tile >= tiles) return;
  W4Block<G, W> blk[U];
  const auto load = [&](int64_t t, int64_t b) {
#pragma unroll
    for (int u = 0; u < U; ++u) blk[u].load(p, t, min<int64_t>(b * U + u, p.kb - 1), lane);
  };
  load(tile, 0);
  for (; tile < tiles; tile += step) {
    float acc[W][RU];
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int r = 0; r < RU; ++r) acc[w][r] = 0.0f;
    for (int64_t b = 0; b < batches; ++b) {
      W4Block<G, W> cur[U];
#pragma unroll
      for (int u = 0; u < U; ++u) cur[u] = blk[u];
      if (b + 1 < batches) load(tile, b + 1);
      else load(min(tile + step, tiles - 1), 0);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (b * U + u < p.kb) {
          half8 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = ld8(xr + (b * U + u) * 128 + 32 * i);
          cur[u].multiply(x, acc, masks);
        }
    }
#pragma unroll
    for (int r = 0; r < RU; ++r) {
      float y[W];
#pragma unroll
      for (int w = 0; w < W; ++w) y[w] = acc[w][r];
      w4Put<F32, W>(p, 4 * r + kq, tile * 16 + a, y);
    }
  }
}

// Some more rows: as w4SplitKernel, 32 rows by 16 columns per workgroup of 8 waves. A weight's operand, scaled before the
// products (exact), serves both blocks of 16 rows, and the sums run through all of the wave's k. Bound by the loads of x, 64
// bytes of each of 16 rows an instruction, which every workgroup makes for itself: 17 / 32 x 2048 x 4096 4.8 / 6.5 us.
template <int G, int W, bool F32>
__global__ __launch_bounds__(512) void w4RowsKernel(W4Params p) {
  const Q4Masks masks;
  constexpr int RB = 2, WAVES = 8, PER = 128 / G;
  __shared__ float red[WAVES][W][RB][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = lane & 15, kq = lane >> 4;
  const int64_t tile = blockIdx.x, m0 = static_cast<int64_t>(blockIdx.y) * 16 * RB;
  const h16* xr[RB];  // rows past M read the last one: their sums are not used
#pragma unroll
  for (int r = 0; r < RB; ++r) xr[r] = p.x + min<int64_t>(m0 + 16 * r + a, p.m - 1) * p.k;
  f32x4 acc[W][RB];
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int r = 0; r < RB; ++r) acc[w][r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t kb = wave; kb < p.kb; kb += WAVES) {
    W4Block<G, W> blk;
    blk.load(p, tile, kb, lane);
    half8 x[RB][4];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t k = kb * 128 + 32 * i + 8 * kq;
        x[r][i] = half8{};
        if (k < p.k) x[r][i] = ld8(xr[r] + k);
      }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned word[4] = {blk.q[w].x, blk.q[w].y, blk.q[w].z, blk.q[w].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h16 f = blk.s[w][i * PER / 4];
        const half8 b = q4Ints(word[i], masks) * half8{f, f, f, f, f, f, f, f};
#pragma unroll
        for (int r = 0; r < RB; ++r) acc[w][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[r][i], b, acc[w][r], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[wave][w][r][e][lane] = acc[w][r][e];
  __syncthreads();
  // accumulator e of block r: row 16 r + 4 (l / 16) + e, column l % 16
  for (int o = threadIdx.x; o < RB * 256; o += 64 * WAVES) {
    const int l = o & 63, e = (o >> 6) & 3, r = o >> 8;
    float y[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      y[w] = 0.0f;
#pragma unroll
      for (int v = 0; v < WAVES; ++v) y[w] += red[v][w][r][e][l];
    }
    w4Put<F32, W>(p, m0 + 16 * r + 4 * (l >> 4) + e, tile * 16 + (l & 15), y);
  }
}

// More rows: workgroup of NW x KG waves, tile BM rows x NW 64 columns (SwiGLU: 32 of the gate's and the up weight's same 32).
// Wave (nw, kg) takes all BM rows of its 64 columns over the k blocks kg, kg + KG, ... of 128 k; the KG sums meet in LDS. x goes
// through LDS, a block ahead in registers; the weights go from memory straight into the registers of the one wave that
// multiplies by them, two tiles' words being the B operands of 32x32x16 MFMAs: a lane's column is l % 32, its k 8 (l / 32) +
// 0 .. 7 of each 16, which are words of lanes 16 (2 c + l / 32) + l % 16 of the column's tile, c the half of the 32 k. They are
// scaled before the product (exact), so the sums run through all k. A block's 8 steps take c = 0 first, so that the next
// block's words of one c are loaded while the other c's are used. Each step's operands are made during the MFMAs of the one
// before.
// 128 x 256 (4 waves side by side, no split): 2048 x 2048 x 6144 of two weights 107 us, 960 TFLOP/s (the library's f16 product of
// the same sizes, without SwiGLU: 102 us); MFMA 51%, VALU 48% of the cycles, two waves a SIMD, the conversion of the codes
// (13 instructions for 8) between them; neither is full, and what keeps the two from overlapping further is not known. 64 x 64
// with 8 k groups, for grids that would leave CUs empty: 409 x 6144 x 2048 23.5 us, 440 TFLOP/s (library 37 us); half of a
// round goes to its start and to joining the sums, x passes the L1 once per 64 columns, and a code is converted for 64 rows
// alone (325 VALU to 32 MFMA instructions per 128 k). 32 x 64: 32 x 2048 x 12288 8.7 us.
template <int BM, int NW, int KG, int G, int W, bool F32>
__global__ __launch_bounds__(64 * NW * KG, 2) void w4GemmKernel(W4Params p) {
  const Q4Masks masks;
  constexpr int RB = BM / 32, THREADS = 64 * NW * KG, PER = 128 / G;
  constexpr int BUF = NW == 1 ? 1 : 2;           // a wave alone orders its own stores and reads
  constexpr int STAGE = BM * 128;                // halves of a k group's block
  constexpr int CH = BM * 16 / (64 * NW);        // its 16-byte chunks per thread of the group
  constexpr int SMEM_A = BUF * KG * STAGE * 2, SMEM_R = KG > 1 ? KG * NW * BM * 64 * 4 : 0;
  __shared__ __attribute__((aligned(16))) char smem[SMEM_A > SMEM_R ? SMEM_A : SMEM_R];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = wave % NW, kg = wave / NW, gt = threadIdx.x - kg * NW * 64;
  const int lr = lane & 31, lh = lane >> 5;
  const GridItem gi = xcdOrderYFast();
  const int64_t m0 = static_cast<int64_t>(gi.y) * BM, c0 = static_cast<int64_t>(gi.x) * NW * (W == 2 ? 32 : 64);
  h16* as = reinterpret_cast<h16*>(smem) + kg * BUF * STAGE;
  // Addresses are a wave-uniform base and a lane's 32-bit offset in bytes. This wave's two blocks of 32 columns:
  const int64_t tiles = (p.n + 15) / 16;
  const char* qb[2];
  const char* sb[2];
  unsigned qo[2], so[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int w = W == 2 ? j : 0;
    const int64_t tile = min<int64_t>((c0 + (W == 2 ? 32 * nw : 64 * nw + 32 * j)) / 16, tiles - 1);
    const unsigned more = ((lane >> 4) & 1) && tile + 1 < tiles ? 1u : 0u;  // the lane's tile is this one or the next
    qb[j] = reinterpret_cast<const char*>(p.q[w] + tile * p.kb * 64);
    sb[j] = reinterpret_cast<const char*>(p.s[w] + tile * p.kb * 16 * PER);
    qo[j] = more * static_cast<unsigned>(p.kb) * 1024u + ((lane & 15) + 16 * lh) * 16;
    so[j] = (more * static_cast<unsigned>(p.kb) * 16u + (lane & 15)) * PER * 2;
  }
  // x: chunk id = gt + 64 NW i -> row id / 16, k 8 (id % 16); 16-byte chunk c of row r lies at slot c ^ (r % 16), so that the
  // rows of a fragment read, one chunk of each, fall on all banks
  const char* xb = reinterpret_cast<const char*>(p.x + m0 * p.k);
  constexpr int RP = 4 * NW;  // rows per chunk of all lanes
  const int xc = 8 * (gt & 15), r0 = gt >> 4, s0 = (gt & 15) ^ (r0 & 15);
  const unsigned xo = static_cast<unsigned>(r0) * static_cast<unsigned>(p.k) * 2u + xc * 2;
  const int last = static_cast<int>(min<int64_t>(p.m - 1 - m0, BM - 1));  // the tile's last row
  // (r0 + i RP) % 16 = r0 % 16 ^ i RP % 16: r0 < RP, a power of two
  const auto slot = [&](int i) { return (r0 + i * RP) * 128 + 8 * (s0 ^ (i * RP & 15)); };
  const int blocks = static_cast<int>((p.kb + KG - 1) / KG);  // of every k group (the last may have one less)
  half8 xr[CH];
  // Block b of this k group starts at k = 128 (kg + b KG). In one that K ends in, a lane whose k lie behind K loads the row's
  // last 8 and stores zeros; rows past M load the last row.
  const auto kOf = [&](int b) { return (kg + static_cast<int64_t>(b) * KG) * 128; };
  const auto xload = [&](int b) {
    const int64_t k = kOf(b);
    if (k + 128 <= p.k && last == BM - 1) {
#pragma unroll
      for (int i = 0; i < CH; ++i)
        xr[i] = *reinterpret_cast<const half8*>(xb + (k + static_cast<int64_t>(i) * RP * p.k) * 2 + xo);
    } else {
      const char* at = xb + min<int64_t>(k + xc, p.k - 8) * 2;
#pragma unroll
      for (int i = 0; i < CH; ++i)
        xr[i] = *reinterpret_cast<const half8*>(at + static_cast<unsigned>(min(r0 + i * RP, last)) * static_cast<unsigned>(p.k) * 2u);
    }
  };
  const auto xstore = [&](int b, int buf) {
    const int64_t k = kOf(b);
    if (k + 128 <= p.k) {
#pragma unroll
      for (int i = 0; i < CH; ++i) st8(as + buf * STAGE + slot(i), xr[i]);
    } else {
      const half8 z = {};
#pragma unroll
      for (int i = 0; i < CH; ++i) st8(as + buf * STAGE + slot(i), k + xc < p.k ? xr[i] : z);
    }
  };
  uint4 q[2][2];  // [column block][c]
  h16 sc[2][PER], scNext[2][PER];
  const auto kbOf = [&](int b) { return min<int64_t>(kg + static_cast<int64_t>(b) * KG, p.kb - 1); };
  const auto wload = [&](int b, int c) {
    const int64_t kb = kbOf(b);
#pragma unroll
    for (int j = 0; j < 2; ++j) q[j][c] = *reinterpret_cast<const uint4*>(qb[j] + kb * 1024 + 512 * c + qo[j]);
  };
  const auto sload = [&](int b, h16 (&s)[2][PER]) {
    const int64_t kb = kbOf(b);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < PER; ++g) s[j][g] = *reinterpret_cast<const h16*>(sb[j] + kb * 32 * PER + so[j] + 2 * g);
  };
  f32x16 acc[RB][2];
#pragma unroll
  for (int i = 0; i < RB; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
  // With one wave to a k group the fences keep the compiler from moving its LDS stores and reads, which are served in
  // order, across each other, and the waves run at their own pace.
  const auto staged = [] {
    if constexpr (NW == 1) {
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  // step t: c = t / 4, 32-k piece i = t % 4 of the block
  const auto operands = [&](const h16* a, int t, half8 (&af)[RB], half8 (&bf)[2]) {
    const int c = t >> 2, i = t & 3;
#pragma unroll
    for (int r = 0; r < RB; ++r) af[r] = ld8(a + (32 * r + lr) * 128 + 8 * ((4 * i + 2 * c + lh) ^ (lr & 15)));
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 v = q[j][c];
      const h16 f = sc[j][32 * i / G];
      bf[j] = q4Ints(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w, masks) * half8{f, f, f, f, f, f, f, f};
    }
  };
  xload(0);
  wload(0, 0);
  wload(0, 1);
  sload(0, sc);
  xstore(0, 0);
  staged();
  for (int b = 0; b < blocks; ++b) {
    const h16* a = as + (BUF == 2 ? b & 1 : 0) * STAGE;
    xload(b + 1);
    sload(b + 1, scNext);
    if (KG == 1 || kg + b * KG < p.kb) {
      half8 af[2][RB], bf[2][2];
      operands(a, 0, af[0], bf[0]);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        if (t < 7) operands(a, t + 1, af[(t + 1) & 1], bf[(t + 1) & 1]);
        if (t == 3) wload(b + 1, 0);
        if (t == 7) wload(b + 1, 1);
#pragma unroll
        for (int i = 0; i < RB; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[t & 1][i], bf[t & 1][j], acc[i][j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int g = 0; g < PER; ++g) sc[j][g] = scNext[j][g];
    if (NW == 1) staged();
    xstore(b + 1, BUF == 2 ? (b + 1) & 1 : 0);
    staged();
  }
  if constexpr (NW == 1 && KG > 1) __syncthreads();  // the sums take the blocks' place
  // What the epilogue adds (bias, residual) is loaded for many outputs at once, before their stores: a load behind a store
  // waits for it.
  const auto in = [&](int64_t row, int64_t col) { return row < p.m && col < p.n; };
  const auto added = [&](int64_t row, int64_t col) {
    if (F32 || !in(row, col)) return static_cast<h16>(0.0f);
    return p.res ? p.res[row * p.n + col] : p.bias ? p.bias[col] : static_cast<h16>(0.0f);
  };
  // Of a bias and a residual together, `added` is the residual; the bias is loaded at its store. They are added in w4Put's order.
  const auto put = [&](int64_t row, int64_t col, float y, h16 add) {
    if (!in(row, col)) return;
    if constexpr (F32) {
      static_cast<float*>(p.out)[row * p.n + col] = y;
    } else {
      if (W == 1 && p.bias && p.res) y += static_cast<float>(p.bias[col]);
      static_cast<h16*>(p.out)[row * p.n + col] = toH16(y + static_cast<float>(add));
    }
  };
  const bool adds = W == 1 && (p.res || p.bias);
  if constexpr (KG == 1) {
    // accumulator r of block (i, j): row 32 i + 8 (r / 4) + 4 lh + r % 4, column lr of column block j
#pragma unroll
    for (int i = 0; i < RB; ++i) {
      h16 add[16][2];
#pragma unroll
      for (int r = 0; r < 16; ++r) add[r][0] = add[r][1] = static_cast<h16>(0.0f);
      if (adds) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            add[r][j] = added(m0 + 32 * i + 8 * (r >> 2) + 4 * lh + (r & 3), c0 + 64 * nw + 32 * j + lr);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t row = m0 + 32 * i + 8 * (r >> 2) + 4 * lh + (r & 3);
        if constexpr (W == 2) {
          put(row, c0 + 32 * nw + lr, siluMul(acc[i][0][r], acc[i][1][r]), add[r][0]);
        } else {
          put(row, c0 + 64 * nw + lr, acc[i][0][r], add[r][0]);
          put(row, c0 + 64 * nw + 32 + lr, acc[i][1][r], add[r][1]);
        }
      }
    }
  } else {
    // 4 columns of a row per item
    constexpr int COLS = W == 2 ? 32 : 64, ALL = NW * BM * COLS / 4, ITEMS = (ALL + THREADS - 1) / THREADS;
    h16 add[ITEMS][4];
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
      const int o = threadIdx.x + t * THREADS, c = o % (COLS / 4) * 4, row = o / (COLS / 4) % BM, v = o / (COLS / 4 * BM);
#pragma unroll
      for (int e = 0; e < 4; ++e) add[t][e] = adds ? added(m0 + row, c0 + v * COLS + c + e) : static_cast<h16>(0.0f);
    }
    float* red = reinterpret_cast<float*>(smem);  // [KG][NW][BM][64]
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          red[(wave * BM + 32 * i + 8 * (r >> 2) + 4 * lh + (r & 3)) * 64 + 32 * j + lr] = acc[i][j][r];
    __syncthreads();
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
      const int o = threadIdx.x + t * THREADS, c = o % (COLS / 4) * 4, row = o / (COLS / 4) % BM, v = o / (COLS / 4 * BM);
      f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f}, u = y;
      if (ALL % THREADS != 0 && o >= ALL) break;
#pragma unroll
      for (int g = 0; g < KG; ++g) {
        const float* at = red + ((g * NW + v) * BM + row) * 64 + c;
        y += *reinterpret_cast<const f32x4*>(at);
        if (W == 2) u += *reinterpret_cast<const f32x4*>(at + 32);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        put(m0 + row, c0 + v * COLS + c + e, W == 2 ? siluMul(y[e], u[e]) : y[e], add[t][e]);
    }
  }
}

}  // namespace lkd

namespace {

bool al16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }
bool groupOk(int g) { return g == 32 || g == 64 || g == 128; }
int launched() { return hipGetLastError() == hipSuccess ? 0 : 2; }
unsigned gridFor(int64_t threads) { return static_cast<unsigned>(std::min<int64_t>((threads + 255) / 256, 65536)); }

int64_t streamLds(const lkd::W4Params& p) { return p.m * (p.kb * 128 + lkd::kStreamPad) * 2; }
bool streamed(const lkd::W4Params& p) { return (p.n + 15) / 16 >= 1536 && streamLds(p) <= 128 << 10; }

template <int RU, int G, int W, bool F32, bool RMS>
void launchFew(const lkd::W4Params& p, hipStream_t s) {
  const int64_t tiles = (p.n + 15) / 16;
  // us, split over 4 / 8 waves against streamed (M = 1, G = 64): K = 2048, N = 4096 3.9 / 4.2 / 6.9; 16384 7.4 / 8.5 / 7.6;
  // 32768 11.2 / 14.2 / 10.3; 65536 19.2 / 27.0 / 16.6; K = 6144, N = 2048 7.3 / 6.2 / 15.4; 8192 9.8 / 10.0 / 15.3; 32768
  // 27.4 / 30.1 / 22.1
  if (streamed(p))
    hipLaunchKernelGGL((lkd::w4StreamKernel<RU, G, W, F32, RMS>), dim3(static_cast<unsigned>(std::min<int64_t>((tiles + 3) / 4, 1024))),
                       dim3(256), static_cast<size_t>(streamLds(p)), s, p);
  else if (p.kb >= 32 && tiles <= 512)
    hipLaunchKernelGGL((lkd::w4SplitKernel<RU, G, W, F32, RMS, 8>), dim3(static_cast<unsigned>(tiles)), dim3(512), 0, s, p);
  else
    hipLaunchKernelGGL((lkd::w4SplitKernel<RU, G, W, F32, RMS, 4>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, s, p);
}

template <int BM, int NW, int KG, int G, int W, bool F32>
void launchGemm(const lkd::W4Params& p, hipStream_t s) {
  constexpr int BN = NW * (W == 2 ? 32 : 64);
  const dim3 grid(static_cast<unsigned>((p.n + BN - 1) / BN), static_cast<unsigned>((p.m + BM - 1) / BM));
  hipLaunchKernelGGL((lkd::w4GemmKernel<BM, NW, KG, G, W, F32>), grid, dim3(64 * NW * KG), 0, s, p);
}

template <int G, int W, bool F32>
void launchRows(const lkd::W4Params& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.n + 15) / 16), static_cast<unsigned>((p.m + 31) / 32));
  hipLaunchKernelGGL((lkd::w4RowsKernel<G, W, F32>), grid, dim3(512), 0, s, p);
}

// A product of M rows by `cols` columns (both weights') on tiles of bm x bn: rounds of the chip's 256 workgroups, each about
// a + K / b us. One round's us at K = 512, 2048, 6144: 32 x 64 5.3, 7.4, 13; 64 x 64 8.0, 10.6, 19; 128 x 256 14, 33, 88.
double w4Us(int64_t m, int64_t cols, int64_t k, int bm, int bn, double a, double b) {
  const int64_t groups = ((m + bm - 1) / bm) * ((cols + bn - 1) / bn);
  return static_cast<double>((groups + 255) / 256) * (a + static_cast<double>(k) / b);
}

// 5 to 16 rows that are not streamed: the split kernel, whose workgroups each read all of x, against 32 x 64 tiles, us at M, K, N
// = 8, 6144, 16384 20 / 16; 16, 6144, 16384 30 / 16; 16, 2048, 12288 9.4 / 8.1; 8, 2048, 12288 6.7 / 8.1; 16, 6144, 2048 9.6 / 12.8.
// Over 16 rows: the rows kernel against 32 x 64 tiles, 32 rows, K, N = 512, 2048 3.2 / 5.3; 2048, 4096 6.5 / 7.3; 4096, 2048
// 9.7 / 9.9 (17 rows 7.3 / 10); 6144, 2048 13.8 / 12.6; 2048, 12288 15 / 8.7.
// The tiles against each other, us of 32 x 64 / 64 x 64 / 128 x 256: M, K, N = 128,
// 2048, 4096 8.1 / 11 / 33; 256, 6144, 2048 14 / 20 / 81; 409, 2048, 2048 14 / 11 / 33; 409, 6144, 2048 26 / 21 / 89; 409,
// 2048, 12288 61 / 57 / 38; 2048, 2048, 2048 57 / 56 / 39; 2048, 2048, 12288 297 / 274 / 109.
template <int G, int W, bool F32>
void launchW4(const lkd::W4Params& p, hipStream_t s) {
  if (p.gamma) return launchFew<1, G, W, F32, true>(p, s);
  if (p.m <= 4) return launchFew<1, G, W, F32, false>(p, s);
  if (p.m <= 16 && (streamed(p) || p.m * ((p.n + 15) / 16) < 8192)) return launchFew<4, G, W, F32, false>(p, s);
  if (p.m > 16 && (p.m + 31) / 32 * ((p.n + 15) / 16) <= 256 && p.k <= 4096) return launchRows<G, W, F32>(p, s);
  const double t32 = w4Us(p.m, p.n * W, p.k, 32, 64, 3.0, 400.0), t64 = w4Us(p.m, p.n * W, p.k, 64, 64, 6.6, 350.0),
               t128 = w4Us(p.m, p.n * W, p.k, 128, 256, 6.0, 65.0);
  if (t32 <= t64 && t32 <= t128) launchGemm<32, 1, 8, G, W, F32>(p, s);
  else if (t64 <= t128) launchGemm<64, 1, 8, G, W, F32>(p, s);
  else launchGemm<128, 4, 1, G, W, F32>(p, s);
}

template <int G>
void launchW4(const lkd::W4Params& p, bool two, bool f32, hipStream_t s) {
  if (two) launchW4<G, 2, false>(p, s);
  else if (f32) launchW4<G, 1, true>(p, s);
  else launchW4<G, 1, false>(p, s);
}

}  // namespace

extern "C" {

int64_t lk_hip_w4_codes_bytes(int64_t n, int64_t k) { return (n + 15) / 16 * ((k + 127) / 128) * 1024; }
int64_t lk_hip_w4_scales_bytes(int64_t n, int64_t k, int group) {
  return groupOk(group) ? (n + 15) / 16 * ((k + 127) / 128) * 16 * (128 / group) * 2 : 0;
}

int lk_hip_w4_quantize(const void* w, void* q, void* s, int64_t n, int64_t k, int group, int nt, void* stream) {
  if (n <= 0 || k <= 0 || !groupOk(group) || !al16(q) || !al16(s)) return 1;
  const lkd::W4Layout p{n, k, (k + 127) / 128, group};
  const unsigned grid = gridFor((n + 15) / 16 * 16 * p.kb * (128 / group));
  hipStream_t st = static_cast<hipStream_t>(stream);
  using lkd::w4QuantizeKernel;
  const auto kernel = group == 32   ? (nt ? w4QuantizeKernel<true, 32> : w4QuantizeKernel<false, 32>)
                      : group == 64 ? (nt ? w4QuantizeKernel<true, 64> : w4QuantizeKernel<false, 64>)
                                    : (nt ? w4QuantizeKernel<true, 128> : w4QuantizeKernel<false, 128>);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, static_cast<const lkd::h16*>(w), static_cast<unsigned*>(q),
                     static_cast<lkd::h16*>(s), p, al16(w) && k % 8 == 0);
  return launched();
}

int lk_hip_w4_pack(const void* codes, const void* scales, void* q, void* s, int* flag, int64_t n, int64_t k, int group,
                   void* stream) {
  if (n <= 0 || k <= 0 || !groupOk(group) || !al16(q) || !al16(s) || n > (int64_t{1} << 36)) return 1;
  const lkd::W4Layout p{n, k, (k + 127) / 128, group};
  const dim3 grid(static_cast<unsigned>((n + 63) / 64), static_cast<unsigned>(std::min<int64_t>(p.kb, 65535)));
  hipLaunchKernelGGL(lkd::w4PackKernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint8_t*>(codes), static_cast<const lkd::h16*>(scales), static_cast<uint4*>(q),
                     static_cast<lkd::h16*>(s), flag, p);
  return launched();
}

int lk_hip_w4_unpack(const void* q, const void* s, void* w, int64_t n, int64_t k, int group, void* stream) {
  if (n <= 0 || k <= 0 || !groupOk(group) || !al16(q) || !al16(s)) return 1;
  const lkd::W4Layout p{n, k, (k + 127) / 128, group};
  hipLaunchKernelGGL(lkd::w4UnpackKernel, dim3(gridFor((k + 7) / 8 * n)), dim3(256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const unsigned*>(q), static_cast<const lkd::h16*>(s), static_cast<lkd::h16*>(w), p);
  return launched();
}

int lk_hip_w4_gemm(const void* x, const void* gamma, const void* q, const void* s, const void* q2, const void* s2,
                   const void* bias, const void* res, void* out, int64_t m, int64_t n, int64_t k, int group, int f32_out,
                   float eps, void* stream) {
  using namespace lkd;
  if (m < 0 || n <= 0 || k <= 0 || k % 8 != 0 || !groupOk(group) || !al16(x) || !al16(q) || !al16(s)) return 1;
  if ((q2 == nullptr) != (s2 == nullptr) || (q2 && (bias || res || f32_out || !al16(q2) || !al16(s2)))) return 1;
  if (f32_out && (bias || res)) return 1;
  if (gamma && (m > 1 || !al16(gamma))) return 1;
  if (m == 0) return 0;
  if (m > 32 * int64_t{65535} || k > (int64_t{1} << 23)) return 1;  // the grid; 32-bit offsets within 128 rows
  const W4Params p{static_cast<const h16*>(x), static_cast<const h16*>(gamma),
                   {static_cast<const uint4*>(q), static_cast<const uint4*>(q2)},
                   {static_cast<const h16*>(s), static_cast<const h16*>(s2)},
                   static_cast<const h16*>(bias), static_cast<const h16*>(res), out, m, n, k, (k + 127) / 128, eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (group == 32) launchW4<32>(p, q2 != nullptr, f32_out != 0, st);
  else if (group == 64) launchW4<64>(p, q2 != nullptr, f32_out != 0, st);
  else launchW4<128>(p, q2 != nullptr, f32_out != 0, st);
  return launched();
}

}  // extern "C"

// ---- registry -----------------------------------------------------------------------------------------------------
namespace lkh {

namespace {

bool w4Shapes(int64_t nt, int64_t kb, int64_t per, int64_t n, int64_t k, int64_t group) {
  return groupOk(static_cast<int>(group)) && nt == (n + 15) / 16 && kb == (k + 127) / 128 && per == 128 / group;
}

// quantize_w4_f16_gpu: w[K, N] (nt: [N, K]) -> q i32[NT, KB, 256], s f16[NT, KB, 16, 128 / G]; attrs group, nt
void runQuantizeW4(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t group = a.ints[9], nt = a.ints[10];
  const int64_t k = a.ints[nt ? 1 : 0], n = a.ints[nt ? 0 : 1];
  LK_REQUIRE(ctx, w4Shapes(a.ints[2], a.ints[3], a.ints[8], n, k, group) && a.ints[4] == 256 && a.ints[7] == 16 &&
                      a.ints[5] == a.ints[2] && a.ints[6] == a.ints[3],
             "quantize_w4: q i32[ceil(N / 16), ceil(K / 128), 256], s f16[.., .., 16, 128 / group], group 32, 64 or 128");
  status(ctx, lk_hip_w4_quantize(a.ptrs[0], a.ptrs[1], a.ptrs[2], n, k, static_cast<int>(group), nt != 0, ctx.stream),
         "quantize_w4: launch failed");
}

// pack_w4_u8_gpu: codes u8[K, N], scales f16[ceil(K / G), N], flag i32[1] (zero; in place) -> q, s; attr group
void runPackW4(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t k = a.ints[0], n = a.ints[1], group = a.ints[12];
  LK_REQUIRE(ctx, w4Shapes(a.ints[5], a.ints[6], a.ints[11], n, k, group) && a.ints[7] == 256 && a.ints[10] == 16 &&
                      a.ints[3] == n && a.ints[2] == (k + group - 1) / group && a.ints[8] == a.ints[5] &&
                      a.ints[9] == a.ints[6] && a.ints[4] == 1,
             "pack_w4: codes u8[K, N], scales f16[ceil(K / group), N], flag i32[1], group 32, 64 or 128");
  status(ctx, lk_hip_w4_pack(a.ptrs[0], a.ptrs[1], a.ptrs[3], a.ptrs[4], P<int>(a, 2), n, k, static_cast<int>(group),
                             ctx.stream),
         "pack_w4: launch failed");
}

// unpack_w4_f16_gpu: q, s -> w f16[K, N]; attr group
void runUnpackW4(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t k = a.ints[7], n = a.ints[8], group = a.ints[9];
  LK_REQUIRE(ctx, n > 0 && k > 0 && w4Shapes(a.ints[0], a.ints[1], a.ints[6], n, k, group) && a.ints[2] == 256,
             "unpack_w4: the weight's q and s, out f16[K, N]");
  status(ctx, lk_hip_w4_unpack(a.ptrs[0], a.ptrs[1], a.ptrs[2], n, k, static_cast<int>(group), ctx.stream),
         "unpack_w4: launch failed");
}

// gemm_w4[_bias|_add|_swiglu]_f16_gpu, rmsnorm_gemm_w4[_swiglu]_f16_gpu (one row), lm_head_w4_f16_gpu:
// x[M, K] [, g[K]], q, s [, q2, s2] [, bias[N] | res[M, N]] -> [M, N]; attr group; float eps with g
enum : int { W4_PLAIN, W4_BIAS, W4_ADD, W4_SWIGLU, W4_LOGITS };
template <int EPI, bool RMS>
void runGemmW4(ExecCtx& ctx, const KernelArgs& a) {
  Ints it(a);
  int ptr = 0;
  const int64_t m = it.next(), k = it.next();
  const void* x = a.ptrs[ptr++];
  const void* g = nullptr;
  if (RMS) {
    g = a.ptrs[ptr++];
    LK_REQUIRE(ctx, it.next() == k, "rmsnorm_gemm_w4: g must be f16[K]");
    LK_REQUIRE(ctx, m == 1, "rmsnorm_gemm_w4: one row (normalize more rows first)");
  }
  const int wts = EPI == W4_SWIGLU ? 2 : 1;
  int64_t dims[2][7];
  const void* q[2] = {nullptr, nullptr};
  const void* s[2] = {nullptr, nullptr};
  for (int w = 0; w < wts; ++w) {
    q[w] = a.ptrs[ptr++];
    s[w] = a.ptrs[ptr++];
    for (int i = 0; i < 7; ++i) dims[w][i] = it.next();
  }
  const void *bias = nullptr, *res = nullptr;
  int64_t e0 = 0, e1 = 0;
  if (EPI == W4_BIAS) {
    bias = a.ptrs[ptr++];
    e0 = it.next();
  } else if (EPI == W4_ADD) {
    res = a.ptrs[ptr++];
    e0 = it.next();
    e1 = it.next();
  }
  const int64_t om = it.next(), n = it.next(), group = it.next();
  for (int w = 0; w < wts; ++w)
    LK_REQUIRE(ctx, w4Shapes(dims[w][0], dims[w][1], dims[w][6], n, k, group) && dims[w][2] == 256 &&
                        dims[w][3] == dims[w][0] && dims[w][4] == dims[w][1] && dims[w][5] == 16,
               "gemm_w4: x f16[M, K], a weight f16[K, N] in 4 bits, group 32, 64 or 128");
  LK_REQUIRE(ctx, om == m && (EPI != W4_BIAS || e0 == n) && (EPI != W4_ADD || (e0 == m && e1 == n)),
             "gemm_w4: out [M, N], bias f16[N], res f16[M, N]");
  status(ctx, lk_hip_w4_gemm(x, g, q[0], s[0], q[1], s[1], bias, res, a.ptrs[ptr], m, n, k, static_cast<int>(group),
                             EPI == W4_LOGITS, F(a, 0, 1e-6f), ctx.stream),
         "gemm_w4: K must be a multiple of 8 and at most 2^23, M at most 2097120, the operands 16-byte aligned");
}

}  // namespace

void registerQ4Kernels() {
  const Device G = Device::Gpu;
  registerKernel({"quantize_w4_f16_gpu", G, runQuantizeW4, 1, 2});
  registerKernel({"pack_w4_u8_gpu", G, runPackW4, 3, 2});
  registerKernel({"unpack_w4_f16_gpu", G, runUnpackW4, 2, 1});
  registerKernel({"gemm_w4_f16_gpu", G, runGemmW4<W4_PLAIN, false>, 3, 1});
  registerKernel({"gemm_w4_bias_f16_gpu", G, runGemmW4<W4_BIAS, false>, 4, 1});
  registerKernel({"gemm_w4_add_f16_gpu", G, runGemmW4<W4_ADD, false>, 4, 1});
  registerKernel({"gemm_w4_swiglu_f16_gpu", G, runGemmW4<W4_SWIGLU, false>, 5, 1});
  registerKernel({"lm_head_w4_f16_gpu", G, runGemmW4<W4_LOGITS, false>, 3, 1});
  registerKernel({"rmsnorm_gemm_w4_f16_gpu", G, runGemmW4<W4_PLAIN, true>, 4, 1});
  registerKernel({"rmsnorm_gemm_w4_swiglu_f16_gpu", G, runGemmW4<W4_SWIGLU, true>, 6, 1});
  registerKernel({"rmsnorm_lm_head_w4_f16_gpu", G, runGemmW4<W4_LOGITS, true>, 4, 1});
}

}  // namespace lkh
