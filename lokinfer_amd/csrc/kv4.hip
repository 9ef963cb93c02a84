// Key / value caches held in 4 bits (lk.ops.q4_gpu; no counterpart in the reference, whose caches are f16 or f32).
//
// A cache is u8 [B, 2, kvh, 72 P] (B sequences; keys, values; P rows, a multiple of 32): per (sequence, key or value, kv
// head) P rows of 64 bytes of codes, then the scales, f16 [4, P], one for each 32 of the head's 128 values (format: q4.h).
// A row whose key or value is not finite is held with NaN key scales and a zero value: a query that sees it gets NaN, one
// that it is masked from is not touched by it.
//
//   lk_hip_kv4_write          k, v f16[B T, kvh 128] to rows pos[b] ..
//   lk_hip_kv4_qknorm_rope    qkv f16[B T, (qh + 2 kvh) 128]: QK-norm and RoPE at positions pos[b] .., q out, k and v written
//   lk_hip_kv4_read           codes and scales -> f16 rows
//   lk_hip_kv4_attention      causal GQA over the cache: query i of sequence b sees rows 0 .. pos[b] + i
//   lk_hip_kv4_reorder        sequence b's rows 0 .. n - 1 become sequence parents[b]'s, in place
#include <algorithm>
#include <cmath>

#include "common.h"
#include "lokinfer_hip.h"
#include "q4.h"

namespace lkd {

constexpr int KHD = 128;

// ---- writing ----------------------------------------------------------------------------------------------------
// 32 lanes quantise a row's key (the first 16, 8 values per lane) and value: the lane's word of codes and its group's scale.
struct Kv4Word {
  unsigned word;
  h16 scale;
};
__device__ __forceinline__ Kv4Word kv4Quantise(half8 x) {
  const int lane = threadIdx.x & 63;
  float v[8], hi = 0.0f, lo = 0.0f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = static_cast<float>(x[e]);
    hi = fmaxf(hi, v[e]);
    lo = fminf(lo, v[e]);
    bad = bad || !(fabsf(v[e]) < INFINITY);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {  // the 4 lanes of a group
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    lo = fminf(lo, __shfl_xor(lo, o, 64));
  }
  const bool rowBad = static_cast<unsigned>(__ballot(bad) >> (lane & 32)) != 0u;
  float s = q4Scale(hi, lo);
  if (rowBad) s = (lane & 16) ? 0.0f : __builtin_nanf("");
  Kv4Word out{0u, static_cast<h16>(s)};
#pragma unroll
  for (int e = 0; e < 8; ++e) out.word |= q4Code(v[e], s) << q4Shift(e);
  return out;
}

// grid: T / 16, kv heads, B. A wave takes 4 rows, two at a time; the scales go through LDS, since a plane's neighbours are
// neighbouring rows'. 32768 rows of 8 heads 62 us (172 MB, 2.8 TB/s; one row per wave and single scales: 108); 409 rows 4.2 us,
// of which 2.5 are a launch's.
constexpr int kWriteRows = 16;
__global__ __launch_bounds__(256) void kv4WriteKernel(char* __restrict__ kv, const h16* __restrict__ k,
                                                      const h16* __restrict__ v, const int64_t* __restrict__ pos, int t,
                                                      int kvh, int64_t cap) {
  __shared__ h16 scales[8][kWriteRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, h = blockIdx.y, seq = blockIdx.z;
  const int first = blockIdx.x * kWriteRows;
  const int64_t p0 = pos[seq];
  char* kb = kv + (static_cast<int64_t>(seq) * 2 * kvh + h) * 72 * cap;
  char* vb = kb + static_cast<int64_t>(kvh) * 72 * cap;
  const auto inside = [&](int i) { return i < t && p0 >= -i && p0 < cap - i; };
  half8 x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int in = first + wave * 4 + 2 * i + (lane >> 5);
    x[i] = half8{};
    if (in < t) x[i] = ld8(((lane & 16) ? v : k) + ((static_cast<int64_t>(seq) * t + in) * kvh + h) * KHD + 8 * l);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int in = wave * 4 + 2 * i + (lane >> 5);
    const Kv4Word y = kv4Quantise(x[i]);
    if (inside(first + in)) *reinterpret_cast<unsigned*>(((lane & 16) ? vb : kb) + (p0 + first + in) * 64 + 4 * l) = y.word;
    if ((l & 3) == 0) scales[(lane & 16) / 4 + (l >> 2)][in] = y.scale;
  }
  __syncthreads();
  const int in = threadIdx.x % kWriteRows, plane = threadIdx.x / kWriteRows;
  if (plane < 8 && inside(first + in))
    *reinterpret_cast<h16*>((plane >= 4 ? vb : kb) + cap * (64 + (plane & 3) * 2) + 2 * (p0 + first + in)) = scales[plane][in];
}

struct Kv4QkrParams {
  const h16* qkv;
  const h16* qg;
  const h16* kg;
  const int64_t* pos;
  char* kv;
  h16* q;
  unsigned rows, t;  // B T
  int64_t cap;
  int qh, kvh;
  float eps;
  RopeTable tab;
};

// One wave per (row, q head) and (row, kv head), grid rows / 4, heads: a q head is normalized and rotated to q, a kv head's key
// likewise and quantised with its value. Arithmetic and roundings of the norm and the rotation as qkRopeKvKernel's. 16 / 8 heads: 1 row 3.8
// us, 409 8.1, 2048 26 (bytes: 6): the sine and cosine of a row's angles in 64 bits, which each of its 24 waves takes for itself.
__global__ __launch_bounds__(256) void kv4QkRopeKernel(Kv4QkrParams p) {
  __shared__ __attribute__((aligned(16))) h16 rows[4][2 * KHD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slot = blockIdx.y;
  const unsigned ri = blockIdx.x * 4 + wave;
  if (ri >= p.rows) return;
  const unsigned seq = ri / p.t;
  const int64_t r = ri, row = p.pos[seq] + (ri - seq * p.t);
  const int64_t width = static_cast<int64_t>(p.qh + 2 * p.kvh) * KHD;
  const bool isQ = slot < p.qh;
  if (!isQ && (row < 0 || row >= p.cap)) return;
  const h16* x = p.qkv + r * width + slot * KHD;
  const h16* g = isQ ? p.qg : p.kg;
  // the loads first, the angle while they are on their way
  const half8 own = lane < KHD / 8 ? ld8(x + 8 * lane) : half8{};  // rowSumSq's piece of a head
  const h16 lo = x[lane], hi = x[lane + 64], glo = g[lane], ghi = g[lane + 64];
  h16 vlo{}, vhi{};
  if (!isQ) {
    const h16* v = x + static_cast<int64_t>(p.kvh) * KHD;
    vlo = v[lane];
    vhi = v[lane + 64];
  }
  float c, s, sum = 0.0f;
  ropeAngle(row, p.tab.invf[lane], c, s);
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(static_cast<float>(own[e]), static_cast<float>(own[e]), sum);
  const float f = rmsFactor(waveSum(sum), KHD, p.eps);
  h16 a, b;
  ropeRotate(static_cast<float>(rmsElem(lo, glo, f)), static_cast<float>(rmsElem(hi, ghi, f)), c, s, a, b);
  if (isQ) {
    h16* o = p.q + r * p.qh * KHD + slot * KHD;
    o[lane] = a;
    o[lane + 64] = b;
    return;
  }
  h16* mine = rows[wave];
  mine[lane] = a;
  mine[lane + 64] = b;
  mine[KHD + lane] = vlo;
  mine[KHD + lane + 64] = vhi;
  // this wave's own slice: its LDS operations complete in order
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int64_t block = 72 * p.cap;
  const Kv4Word y = kv4Quantise(ld8(mine + 8 * (lane & 31)));  // the upper lanes as the lower ones
  if (lane >= 32) return;
  char* at = p.kv + (static_cast<int64_t>(seq) * 2 * p.kvh + (slot - p.qh) + (lane < 16 ? 0 : p.kvh)) * block;
  const int l = lane & 15;
  *reinterpret_cast<unsigned*>(at + row * 64 + 4 * l) = y.word;
  if ((l & 3) == 0) *reinterpret_cast<h16*>(at + p.cap * 64 + (l >> 2) * 2 * p.cap + 2 * row) = y.scale;
}

// ---- reading ----------------------------------------------------------------------------------------------------
// one thread per 8 values, grid cap 16 / 256, blocks: blocks of 72 cap bytes -> f16 [blocks, cap, 128]; HBM-bound, 512 blocks of
// 1216 rows 35 us (204 MB, 5.8 TB/s)
__global__ __launch_bounds__(256) void kv4ReadKernel(const char* __restrict__ kv, h16* __restrict__ out, int64_t blocks,
                                                     unsigned cap) {
  const Q4Masks masks;
  for (int64_t blk = blockIdx.y; blk < blocks; blk += gridDim.y) {
    const char* at = kv + blk * 72 * cap;
    h16* o = out + blk * cap * KHD;
    for (unsigned id = blockIdx.x * 256 + threadIdx.x; id < cap * 16; id += gridDim.x * 256) {
      const unsigned row = id >> 4, w = id & 15;
      const h16 s = *reinterpret_cast<const h16*>(at + static_cast<int64_t>(cap) * (64 + (w >> 2) * 2) + 2 * row);
      const half8 v = q4Ints(*reinterpret_cast<const unsigned*>(at + static_cast<int64_t>(id) * 4), masks);
      st8(o + static_cast<int64_t>(id) * 8, v * half8{s, s, s, s, s, s, s, s});
    }
  }
}

// ---- attention ----------------------------------------------------------------------------------------------------
struct Kv4Params {
  const h16* q;  // [B T, qh 128]
  const char* kv;
  const int64_t* pos;
  h16* out;
  float* part;  // [B T qh, splits, 130]: (max, sum, out[128]) of each workgroup's keys
  int64_t cap;
  unsigned t, blocks;          // blocks: row blocks of a kv head
  int qh, kvh, group, splits;  // group = qh / kvh
  float scale;  // log2(e) / sqrt(128)
  unsigned long long* err;
};

// 16 RB rows of a kv head per workgroup of KW waves: row r = i group + h (query i's q heads side by side). A wave takes 64 keys
// at a time, four tiles of 16, on 16x16x32 MFMAs, each operand of the cache made once for the RB blocks of 16 rows:
// S = K Q^T: lane (key l % 16, kq = l / 16) loads 16 bytes of its key's row, the codes of scale group kq; its word w, scaled
// (exact in f16), is the A operand of step w, dims 32 kq + 8 w .., the B operand row l % 16's same dims. Its accumulators are
// then row l % 16's scores of keys 4 kq + 0 .. 3, on which the softmax runs in f32 (log2 units).
// O^T = V^T P^T over two tiles: the lane's own 8 weights are the B operand as they are, as two f16 parts, hi and lo = p - hi.
// f16's smallest step is 2^-24, so the pair is off by 2^-22 of p or by 2^-25, and by 2^-37 of the row's largest weight, which is
// held at 2^12 or above (kStart). The A operand is 8 keys of one dim: lane (db = l % 16, kq) loads those keys' words
// db, dims 8 db .. 8 db + 7; the low halves of two keys' words put side by side hold the even dims' codes as pairs, the high
// halves the odd ones', so each dim's operand is masked out of them as a row's codes are out of a word.
// Chunks are dealt over the waves of all workgroups of a row block (splits); the waves' sums meet in LDS.
// Keys from the longest row's end on have their weight and their value's scale set to zero, whatever the memory holds there.
// A row's weights are 2^(score - m): m is set 12 below a maximum, and again, with its sums rescaled, only where a score exceeds
// it by 15 (2^15 fits f16), since nearly every tile brings some row a slightly larger score. m 7 below a maximum takes up to 1.6%
// less time, m at one with room for 2^8 up to 2.3%, which loses weights under 2^-25 of the largest. A score is one fma away
// from m, its product with the scale not rounded by itself; where f32's steps are too coarse for that, from 2^20 on (at 2^28 the
// difference would leave f16), the product is rounded first, as the maximum's was, and m is the maximum: 1% of the time.
// 16 / 8 heads: one query over 417 rows 6.7 us and over 32768 12.3 + 4.2 of the joining launch (38 MB, 2.3 TB/s): latency, of one
// chunk in the first; its 128 registers (4 waves a SIMD) leave 4 values in scratch. 2048 queries over as many rows 46 us, 370
// TFLOP/s: bound by VALU (some 70% of the cycles, MFMA 28%), half of it the codes' conversion, which 32 rows share, half the
// softmax. Tiles of f16 made once per call and shared through LDS took 6 + 50; more rows a wave leave one wave a SIMD (61 us).
constexpr float kTop = 15.0f, kStart = 12.0f, kCoarse = 0x1p20f;
template <int RB, int KW>
__global__ __launch_bounds__(64 * KW) __attribute__((amdgpu_waves_per_eu(RB == 1 ? 4 : 2))) void kv4AttnKernel(Kv4Params p) {
  const Q4Masks masks;
  constexpr int ROWS = 16 * RB;
  __shared__ __attribute__((aligned(16))) float os[KW][ROWS][KHD + 4];
  __shared__ float ms[KW][ROWS], ls[KW][ROWS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lc = lane & 15, kq = lane >> 4;
  const unsigned group = static_cast<unsigned>(p.group), rowsHead = p.t * group;
  // with 8 kv heads one XCD's L2 each; the last rows, which see the most keys, first
  const unsigned kvHead = blockIdx.x % static_cast<unsigned>(p.kvh), rest = blockIdx.x / static_cast<unsigned>(p.kvh);
  const unsigned split = rest % static_cast<unsigned>(p.splits), rb = p.blocks - 1 - rest / static_cast<unsigned>(p.splits);
  const int64_t seq = blockIdx.y;
  const int64_t p0 = p.pos[seq];
  const int cap = static_cast<int>(p.cap);
  // rows of the cache that query i sees; the block's last and first row's
  const auto sees = [&](int64_t i) { return p0 < 0 ? 0 : static_cast<int>(p0 < p.cap ? min<int64_t>(p0 + i + 1, p.cap) : p.cap); };
  const int nk = sees(min(rb * ROWS + ROWS - 1, rowsHead - 1) / group), nkAll = sees(rb * ROWS / group);
  half8 qf[RB][4];
  int nkRow[RB];
#pragma unroll
  for (int k = 0; k < RB; ++k) {
    const unsigned row = min(rb * ROWS + 16 * k + lc, rowsHead - 1), qi = row / group;
    nkRow[k] = sees(qi);
    const h16* q = p.q + ((seq * p.t + qi) * p.qh + kvHead * group + (row - qi * group)) * KHD + 32 * kq;
#pragma unroll
    for (int w = 0; w < 4; ++w) qf[k][w] = ld8(q + 8 * w);
  }
  if (rest == 0 && kvHead == 0 && threadIdx.x == 0 && (p0 < 0 || p0 > p.cap - p.t))
    raiseDeviceError(p.err, LK_DEVERR_POSITION, p0 < 0 || p0 > p.cap ? p0 : p0 + p.t - 1);
  const int64_t block = 72 * p.cap;
  const char* kb = p.kv + (seq * 2 * p.kvh + kvHead) * block;
  const char* vb = kb + p.kvh * block;
  // a chunk's base is uniform, a lane's place in it a 32-bit offset in bytes: codes and scales of keys and values
  const unsigned kOff = lc * 64 + 16 * kq, vOff = 4 * kq * 64 + 4 * lc;
  const unsigned ksOff = kq * static_cast<unsigned>(cap) * 2 + lc * 2, vsOff = (lc >> 2) * static_cast<unsigned>(cap) * 2 + 8 * kq;
  const int chunks = (nk + 63) / 64, step = p.splits * KW;
  f32x4 acc[RB][8];
  float m[RB];   // what is taken off a row's scores: the maximum it was set at times the scale, rounded once, less kStart
  f32x4 l[RB];   // the weights' sum, four times: a product with ones
  const h16 one = static_cast<h16>(1.0f);
  const half8 ones{one, one, one, one, one, one, one, one};
#pragma unroll
  for (int k = 0; k < RB; ++k) {
    m[k] = -INFINITY;
    l[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[k][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int c = static_cast<int>(split) * KW + wave; c < chunks; c += step) {
    // Rows behind the last key are read as they lie, and masked below; the cache ends with a chunk or in its middle, where
    // the second half reads the first's rows.
    const int64_t half = c * 64 + 32 < cap ? 32 : 0, c0 = static_cast<int64_t>(c) * 64;
    uint4 kw[4];
    h16 ks[4];
    unsigned vw[4][4];
    half4 vs[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t r0 = c0 + (u >> 1) * half;
      kw[u] = *reinterpret_cast<const uint4*>(kb + r0 * 64 + kOff + 1024 * (u & 1));
      ks[u] = *reinterpret_cast<const h16*>(kb + 64 * p.cap + r0 * 2 + ksOff + 32 * (u & 1));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t r0 = c0 + (u >> 1) * half;
#pragma unroll
      for (int r = 0; r < 4; ++r) vw[u][r] = *reinterpret_cast<const unsigned*>(vb + r0 * 64 + vOff + 1024 * (u & 1) + 64 * r);
      vs[u] = *reinterpret_cast<const half4*>(vb + 64 * p.cap + r0 * 2 + vsOff + 32 * (u & 1));
    }
    f32x4 s[RB][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned w4[4] = {kw[u].x, kw[u].y, kw[u].z, kw[u].w};
      const h16 f = ks[u];
#pragma unroll
      for (int k = 0; k < RB; ++k) s[k][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const half8 a = q4Ints(w4[w], masks) * half8{f, f, f, f, f, f, f, f};
#pragma unroll
        for (int k = 0; k < RB; ++k) s[k][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[k][w], s[k][u], 0, 0, 0);
      }
    }
    if (c * 64 + 64 > nkAll) {  // keys past some row's
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = c * 64 + 16 * u + 4 * kq + r;
#pragma unroll
          for (int k = 0; k < RB; ++k)
            if (key >= nkRow[k]) s[k][u][r] = -INFINITY;
          if (key >= nk) vs[u][r] = static_cast<h16>(0.0f);
        }
    }
    half8 ph[RB][2], pl[RB][2];
#pragma unroll
    for (int k = 0; k < RB; ++k) {
      float mx = s[k][0][0];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[k][u][r]);
      mx = crossRowMax(mx) * p.scale;
      if (__any(mx - m[k] > kTop)) {
        const bool grows = mx - m[k] > kTop;  // (each row by itself: its sums do not depend on its neighbours)
        const float to = fabsf(mx) > kCoarse ? mx : mx - kStart, corr = grows ? __builtin_amdgcn_exp2f(m[k] - to) : 1.0f;
        l[k] *= corr;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[k][e] *= corr;
        m[k] = grows ? to : m[k];
      }
      float sc = p.scale;
      if (__any(fabsf(mx) > kCoarse)) {
        const bool coarse = fabsf(mx) > kCoarse;
        sc = coarse ? 1.0f : sc;
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[k][u][r] = coarse ? s[k][u][r] * p.scale : s[k][u][r];
      }
      const float base = m[k] == -INFINITY ? 0.0f : m[k];  // no key so far: every weight 0 (or a NaN kept)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          typedef float f32x2 __attribute__((ext_vector_type(2)));
          const f32x2 e = {__builtin_amdgcn_exp2f(fmaf(s[k][u][r], sc, -base)),
                           __builtin_amdgcn_exp2f(fmaf(s[k][u][r + 1], sc, -base))};
          const half2v hi = __builtin_convertvector(e, half2v);
          const half2v lo = __builtin_convertvector((f32x2{fmaf(static_cast<float>(hi[0]), -1.0f, e[0]),
                                                           fmaf(static_cast<float>(hi[1]), -1.0f, e[1])}), half2v);
          const int at = 4 * (u & 1) + r;
          ph[k][u >> 1][at] = hi[0];
          ph[k][u >> 1][at + 1] = hi[1];
          pl[k][u >> 1][at] = lo[0];
          pl[k][u >> 1][at + 1] = lo[1];
        }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        l[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, ph[k][t], l[k], 0, 0, 0);
        l[k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[k][t], l[k], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {  // keys 32 t ..: tiles 2 t, 2 t + 1
      unsigned even[4], odd[4];
      half2v sc[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // keys 2 j, 2 j + 1 of the lane's 8
        const unsigned a = vw[2 * t + (j >> 1)][2 * (j & 1)], b = vw[2 * t + (j >> 1)][2 * (j & 1) + 1];
        even[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        odd[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        sc[j] = half2v{vs[2 * t + (j >> 1)][2 * (j & 1)], vs[2 * t + (j >> 1)][2 * (j & 1) + 1]};
      }
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        half2v dims[4][4];  // [dim 2 i + o][pair of keys]
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const half8 v = q4Ints(o ? odd[j] : even[j], masks);
#pragma unroll
          for (int i = 0; i < 4; ++i) dims[i][j] = half2v{v[2 * i], v[2 * i + 1]} * sc[j];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const half8 a{dims[i][0][0], dims[i][0][1], dims[i][1][0], dims[i][1][1],
                        dims[i][2][0], dims[i][2][1], dims[i][3][0], dims[i][3][1]};
#pragma unroll
          for (int k = 0; k < RB; ++k) {
            acc[k][2 * i + o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[k][t], acc[k][2 * i + o], 0, 0, 0);
            acc[k][2 * i + o] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[k][t], acc[k][2 * i + o], 0, 0, 0);
          }
        }
      }
    }
  }
  // accumulator r of dim e: dim 8 (4 kq + r) + e of row l % 16
  const int rows = static_cast<int>(min(rowsHead - rb * ROWS, static_cast<unsigned>(ROWS)));
#pragma unroll
  for (int k = 0; k < RB; ++k) {
    const int row = 16 * k + lc;
    if (row < rows) {
      if (kq == 0) {
        ms[wave][row] = m[k];
        ls[wave][row] = l[k][0];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float* o = &os[wave][row][8 * (4 * kq + r)];
        *reinterpret_cast<f32x4*>(o) = f32x4{acc[k][0][r], acc[k][1][r], acc[k][2][r], acc[k][3][r]};
        *reinterpret_cast<f32x4*>(o + 4) = f32x4{acc[k][4][r], acc[k][5][r], acc[k][6][r], acc[k][7][r]};
      }
    }
  }
  __syncthreads();
  // 4 dims of a row per item
  for (int o = threadIdx.x; o < rows * (KHD / 4); o += 64 * KW) {
    const int r = o / (KHD / 4), d = o % (KHD / 4) * 4;
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w) mm = fmaxf(mm, ms[w][r]);
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float f = ms[w][r] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms[w][r] - mm);  // no key: zeros, or a NaN
      ll = fmaf(f, ls[w][r], ll);
      const f32x4 part = *reinterpret_cast<const f32x4*>(&os[w][r][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(f, part[e], y[e]);
    }
    const unsigned i = (rb * ROWS + r) / group;
    const int64_t at = (seq * p.t + i) * p.qh + kvHead * group + (rb * ROWS + r - i * group);
    if (p.splits == 1) {
      const bool noRow = p0 < 0 || p0 >= p.cap - i;
      half4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = noRow ? static_cast<h16>(__builtin_nanf("")) : toH16(y[e] / ll);
      *reinterpret_cast<half4*>(p.out + at * KHD + d) = out;
    } else {
      float* pp = p.part + (at * p.splits + split) * (KHD + 2);
      *reinterpret_cast<float2*>(pp + 2 + d) = make_float2(y[0], y[1]);
      *reinterpret_cast<float2*>(pp + 4 + d) = make_float2(y[2], y[3]);
      if (d == 0) *reinterpret_cast<float2*>(pp) = make_float2(mm, ll);
    }
  }
}

// one workgroup per (q head, query): the splits' partials, 32 at a time, all loads in flight together: 4 us, a launch and one
// latency
__global__ __launch_bounds__(128) void kv4MergeKernel(Kv4Params p) {
  const int d = threadIdx.x;
  const unsigned qi = blockIdx.y, seq = qi / p.t;
  const int64_t at = static_cast<int64_t>(qi) * p.qh + blockIdx.x, p0 = p.pos[seq];
  const bool noRow = p0 < 0 || p0 >= p.cap - (qi - seq * p.t);
  const float* part = p.part + at * p.splits * (KHD + 2);
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int s0 = 0; s0 < p.splits; s0 += 32) {
    float mc[32], lc[32], oc[32], mb = m;
#pragma unroll
    for (int s = 0; s < 32; ++s) {
      const bool in = s0 + s < p.splits;
      const float* pp = part + (in ? s0 + s : 0) * (KHD + 2);
      mc[s] = in ? pp[0] : -INFINITY;
      lc[s] = in ? pp[1] : 0.0f;
      oc[s] = in ? pp[2 + d] : 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 32; ++s) mb = fmaxf(mb, mc[s]);
    const float corr = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mb);
    l *= corr;
    o *= corr;
#pragma unroll
    for (int s = 0; s < 32; ++s) {
      const float f = mc[s] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mc[s] - mb);  // no key: zeros, or a NaN
      l = fmaf(f, lc[s], l);
      o = fmaf(f, oc[s], o);
    }
    m = mb;
  }
  p.out[at * KHD + d] = noRow ? static_cast<h16>(__builtin_nanf("")) : toH16(o / l);
}

// ---- moving caches between sequences ------------------------------------------------------------------------------
// One thread per 16 bytes of codes or of a scale plane (2 bytes behind its last whole 8 rows) of a (layer, key or value, kv
// head)'s live rows: it reads the piece of the parent of every sequence whose parent is another, then writes them, so that no
// write comes before a read of the same bytes. MB: B rounded up, so that the pieces stay in registers, all reads in flight
// together. HBM-bound: 2 layers of 16 sequences of 1100 rows 20 us (81 MB read and written, 4.0 TB/s), of 4 of 448 rows 4.3.
constexpr int kMaxBeams = 32;
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <int MB, typename T>
__device__ __forceinline__ void kv4Move(char* at, int64_t seqStride, const int64_t* __restrict__ parents, int b, T none) {
  T v[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    v[i] = none;
    const int64_t from = i < b ? parents[i] : i;
    if (from != i && from >= 0 && from < b) v[i] = *reinterpret_cast<const T*>(at + from * seqStride);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
    if (i < b && parents[i] != i) *reinterpret_cast<T*>(at + i * seqStride) = v[i];
}

template <int MB>
__global__ __launch_bounds__(256) void kv4ReorderKernel(char* __restrict__ kv, const int64_t* __restrict__ parents,
                                                        const int64_t* __restrict__ n, int64_t layers, int b, int kvh,
                                                        int64_t cap, unsigned long long* err) {
  const int64_t rows = min(max<int64_t>(*n, 0), cap), blk = blockIdx.y, layer = blk / (2 * kvh), in = blk - layer * 2 * kvh;
  const int64_t seqStride = 2 * kvh * 72 * cap;
  char* base = kv + layer * b * seqStride + in * 72 * cap;
  if (blockIdx.x == 0 && blk == 0 && threadIdx.x == 0) {
    if (*n < 0 || *n > cap) raiseDeviceError(err, LK_DEVERR_POSITION, *n);
    for (int i = 0; i < b; ++i)
      if (parents[i] < 0 || parents[i] >= b) raiseDeviceError(err, LK_DEVERR_INDEX, parents[i]);
  }
  const int64_t whole = rows / 8, rest = rows - whole * 8, codes = rows * 4, items = codes + 4 * (whole + rest);
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < items;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    constexpr unsigned kNan2 = 0x7E007E00u;  // where a parent is not there
    if (id < codes + 4 * whole) {
      int64_t at = id * 16;
      if (id >= codes) {
        const int64_t j = id - codes, g = j / whole;
        at = 64 * cap + g * 2 * cap + 16 * (j - g * whole);
      }
      kv4Move<MB>(base + at, seqStride, parents, b, u32x4{kNan2, kNan2, kNan2, kNan2});
    } else {
      const int64_t j = id - codes - 4 * whole, g = j / rest;
      kv4Move<MB, unsigned short>(base + 64 * cap + g * 2 * cap + 16 * whole + 2 * (j - g * rest), seqStride, parents, b,
                                  kNan2 & 0xFFFFu);
    }
  }
}

}  // namespace lkd

namespace {

bool al16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }
int launched() { return hipGetLastError() == hipSuccess ? 0 : 2; }
constexpr int64_t kMostRows = int64_t{1} << 27;  // of a cache: a row's 16 words and a chunk of 64 rows fit 32 bits
bool kvOk(const void* kv, int64_t b, int kvh, int64_t cap) {
  return b > 0 && kvh > 0 && kvh <= 65535 && cap > 0 && cap % 32 == 0 && cap <= kMostRows && al16(kv);
}
// rows of a call: they are counted in 32 bits
bool rowsOk(int64_t b, int64_t t) { return t >= 0 && t <= 0x7FFFFFFF && b <= 65535 && b * t <= 0x7FFFFFFF; }

// Row blocks and waves of a workgroup. us of (1, 8) / (1, 4) / (2, 8) / (2, 4) by T queries over P rows, 16 / 8 heads: 256, 512
// 8.1 / 8.1 / 11 / 10; 512, 512 11 / 9.9 / 11 / 11; 1024, 1024 24 / 23 / 23 / 20; 300, 2048 27 / 28 / 22 / 23; 600, 2048 37 / 37 /
// 37 / 35; 2048, 2048 61 / 60 / 57 / 46; 2048, 8192 307 / 316 / 244 / 235; 256, 32768 194 / 237 / 241 / 294; 409, 32768 329 /
// 350 / 250 / 295.
struct Kv4Shape {
  int rb, kw;
};
Kv4Shape kv4Shape(int64_t b, int64_t rows, int kvh, int64_t cap) {
  const int64_t groups = b * kvh * ((rows + 15) / 16);
  if (groups <= 256) return {1, 8};
  if (groups <= 640 && cap <= 1024) return {1, 4};
  return groups <= 640 ? Kv4Shape{2, 8} : Kv4Shape{2, 4};
}

// Workgroups over a row block's keys: one for up to 1024 rows (a launch more costs 4 us), else the chip's 256 in all, of at
// least 512 rows each. p32768 at 16 / 8 heads, 16 / 32 / 64 of them: 21 / 17 / 20 us with the joining launch.
int kv4Splits(int64_t b, int64_t t, int qh, int kvh, int64_t cap) {
  const int64_t groups = b * kvh * ((t * (qh / kvh) + 15) / 16);
  if (cap <= 1024 || groups >= 256) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((cap + 511) / 512, 256 / groups)));
}

}  // namespace

extern "C" {

int lk_hip_kv4_write(void* kv, const void* k, const void* v, const int64_t* pos, int64_t b, int64_t t, int kvh, int64_t cap,
                     void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || !rowsOk(b, t) || !al16(k) || !al16(v)) return 1;
  if (t == 0) return 0;
  const dim3 grid(static_cast<unsigned>((t + kWriteRows - 1) / kWriteRows), static_cast<unsigned>(kvh), static_cast<unsigned>(b));
  hipLaunchKernelGGL(kv4WriteKernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<char*>(kv),
                     static_cast<const h16*>(k), static_cast<const h16*>(v), pos, static_cast<int>(t), kvh, cap);
  return launched();
}

int lk_hip_kv4_qknorm_rope(const void* qkv, const void* qg, const void* kg, const int64_t* pos, void* kv, void* q, int64_t b,
                           int64_t t, int qh, int kvh, int64_t cap, float eps, float theta, void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || !rowsOk(b, t) || qh <= 0 || !al16(qkv)) return 1;
  if (t == 0) return 0;
  if (qh + kvh > 65535) return 1;
  Kv4QkrParams p{static_cast<const h16*>(qkv), static_cast<const h16*>(qg), static_cast<const h16*>(kg), pos,
                 static_cast<char*>(kv), static_cast<h16*>(q), static_cast<unsigned>(b * t), static_cast<unsigned>(t), cap, qh, kvh,
                 eps, {}};
  for (int j = 0; j < 64; ++j) p.tab.invf[j] = 1.0f / std::pow(theta, static_cast<float>(2 * j) / 128.0f);
  hipLaunchKernelGGL(kv4QkRopeKernel, dim3(static_cast<unsigned>((b * t + 3) / 4), static_cast<unsigned>(qh + kvh)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return launched();
}

int lk_hip_kv4_read(const void* kv, void* out, int64_t blocks, int64_t cap, void* stream) {
  using namespace lkd;
  if (blocks < 0 || cap <= 0 || cap % 32 != 0 || cap > kMostRows || !al16(kv) || !al16(out)) return 1;
  if (blocks == 0) return 0;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(cap / 16, 256)), static_cast<unsigned>(std::min<int64_t>(blocks, 65535)));
  hipLaunchKernelGGL(kv4ReadKernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const char*>(kv),
                     static_cast<h16*>(out), blocks, static_cast<unsigned>(cap));
  return launched();
}

int64_t lk_hip_kv4_attention_workspace_bytes(int64_t b, int64_t t, int qh, int kvh, int64_t cap) {
  if (b <= 0 || t <= 0 || qh <= 0 || kvh <= 0 || qh % kvh != 0 || cap <= 0) return 0;
  const int64_t s = kv4Splits(b, t, qh, kvh, cap);
  return s > 1 ? s * b * t * qh * (lkd::KHD + 2) * 4 : 0;
}

int lk_hip_kv4_attention(const void* q, const void* kv, const int64_t* pos, void* out, int64_t b, int64_t t, int qh, int kvh,
                         int64_t cap, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || !rowsOk(b, t) || qh <= 0 || qh % kvh != 0 || !al16(q) || !al16(out)) return 1;
  if (t == 0) return 0;
  const int64_t need = lk_hip_kv4_attention_workspace_bytes(b, t, qh, kvh, cap);
  if (need > 0 && (!workspace || workspace_bytes < need || !al16(workspace))) return 3;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int splits = kv4Splits(b, t, qh, kvh, cap);
  const int64_t rows = t * (qh / kvh);
  const Kv4Shape shape = kv4Shape(b, rows, kvh, cap);
  const int64_t blocks = (rows + 16 * shape.rb - 1) / (16 * shape.rb);
  if (rows > 0x7FFFFFFF || blocks * splits * kvh > 0x7FFFFFFF || (splits > 1 && b * t > 65535)) return 1;
  const Kv4Params p{static_cast<const h16*>(q), static_cast<const char*>(kv), pos, static_cast<h16*>(out),
                    static_cast<float*>(workspace), cap, static_cast<unsigned>(t), static_cast<unsigned>(blocks), qh, kvh,
                    qh / kvh, splits, kLog2e / std::sqrt(static_cast<float>(KHD)), lkh::deviceErrorRecord()};
  const dim3 grid(static_cast<unsigned>(blocks * splits * kvh), static_cast<unsigned>(b));
  const auto kernel = shape.rb == 1 ? (shape.kw == 8 ? kv4AttnKernel<1, 8> : kv4AttnKernel<1, 4>)
                                    : (shape.kw == 8 ? kv4AttnKernel<2, 8> : kv4AttnKernel<2, 4>);
  hipLaunchKernelGGL(kernel, grid, dim3(64 * shape.kw), 0, s, p);
  if (splits > 1)
    hipLaunchKernelGGL(kv4MergeKernel, dim3(static_cast<unsigned>(qh), static_cast<unsigned>(b * t)), dim3(128), 0, s, p);
  return launched();
}

int lk_hip_kv4_reorder(void* kv, const int64_t* parents, const int64_t* n, int64_t layers, int64_t b, int kvh, int64_t cap,
                       void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || layers < 0 || b > kMaxBeams || layers * 2 * kvh > 65535) return 1;
  if (layers == 0) return 0;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((cap * 9 / 2 + 255) / 256, 64)),
                  static_cast<unsigned>(layers * 2 * kvh));
  const auto kernel = b <= 4 ? kv4ReorderKernel<4> : b <= 8 ? kv4ReorderKernel<8> : b <= 16 ? kv4ReorderKernel<16>
                                                                                         : kv4ReorderKernel<32>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<char*>(kv), parents, n, layers,
                     static_cast<int>(b), kvh, cap, lkh::deviceErrorRecord());
  return launched();
}

}  // extern "C"

// ---- registry -----------------------------------------------------------------------------------------------------
namespace lkh {

namespace {

bool kv4Layout(int64_t two, int64_t bytes) { return two == 2 && bytes > 0 && bytes % (72 * 32) == 0; }

// kv4_write_f16_gpu: kv u8[B, 2, kvh, 72 P], k, v f16[B T, kvh 128], pos i64[B] (in place)
void runKv4Write(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t b = a.ints[0], kvh = a.ints[2], cap = a.ints[3] / 72, rows = a.ints[4];
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Layout(a.ints[1], a.ints[3]) && rows % b == 0 && a.ints[5] == kvh * 128 &&
                      a.ints[6] == rows && a.ints[7] == a.ints[5] && a.ints[8] == b,
             "kv4_write: kv u8[B, 2, kvh, 72 P] with P % 32 == 0, k and v f16[B T, kvh 128], pos i64[B]");
  status(ctx, lk_hip_kv4_write(a.ptrs[0], a.ptrs[1], a.ptrs[2], P<int64_t>(a, 3), b, rows / b, static_cast<int>(kvh), cap,
                               ctx.stream),
         "kv4_write: kv, k and v must be 16-byte aligned, B at most 65535, P at most 2^27");
}

// qknorm_rope_kv4_f16_gpu: qkv f16[B T, (qh + 2 kvh) 128], qg, kg f16[128], pos i64[B], kv (in place) -> q f16[B T, qh 128];
// floats eps, theta
void runKv4Qkr(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t rows = a.ints[0], b = a.ints[4], kvh = a.ints[7], cap = a.ints[8] / 72, qw = a.ints[10];
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Layout(a.ints[6], a.ints[8]) && a.ints[5] == b && rows % b == 0 &&
                      a.ints[2] == 128 && a.ints[3] == 128 && qw > 0 && qw % 128 == 0 &&
                      a.ints[1] == qw + 2 * kvh * 128 && a.ints[9] == rows,
             "qknorm_rope_kv4: qkv f16[B T, (qh + 2 kvh) 128], gains f16[128], pos i64[B], kv u8[B, 2, kvh, 72 P]");
  status(ctx, lk_hip_kv4_qknorm_rope(a.ptrs[0], a.ptrs[1], a.ptrs[2], P<int64_t>(a, 3), a.ptrs[4], a.ptrs[5], b, rows / b,
                                     static_cast<int>(qw / 128), static_cast<int>(kvh), cap, F(a, 0, 1e-6f), F(a, 1, 1e6f),
                                     ctx.stream),
         "qknorm_rope_kv4: qkv and kv must be 16-byte aligned, B and heads at most 65535, P at most 2^27");
}

// kv4_read_f16_gpu: kv u8[blocks, 72 P] -> f16[blocks, P, 128]
void runKv4Read(ExecCtx& ctx, const KernelArgs& a) {
  LK_REQUIRE(ctx, kv4Layout(2, a.ints[1]) && a.ints[2] == a.ints[0] && a.ints[3] == a.ints[1] / 72 && a.ints[4] == 128,
             "kv4_read: kv u8[blocks, 72 P] with P % 32 == 0, out f16[blocks, P, 128]");
  status(ctx, lk_hip_kv4_read(a.ptrs[0], a.ptrs[1], a.ints[0], a.ints[3], ctx.stream), "kv4_read: kv must be 16-byte aligned, P at most 2^27");
}

// attention_kv4_f16_gpu: q f16[B T, qh 128], kv u8[B, 2, kvh, 72 P], pos i64[B] -> out f16[B T, qh 128], work f32[n]
void runKv4Attention(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t rows = a.ints[0], width = a.ints[1], b = a.ints[2], kvh = a.ints[4], cap = a.ints[5] / 72;
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Layout(a.ints[3], a.ints[5]) && rows % b == 0 && width > 0 &&
                      width % (128 * kvh) == 0 && a.ints[6] == b && a.ints[7] == rows && a.ints[8] == width,
             "attention_kv4: q f16[B T, qh 128], kv u8[B, 2, kvh, 72 P], qh a multiple of kvh, pos i64[B]");
  const int rc = lk_hip_kv4_attention(a.ptrs[0], a.ptrs[1], P<int64_t>(a, 2), a.ptrs[3], b, rows / b,
                                      static_cast<int>(width / 128), static_cast<int>(kvh), cap, a.ptrs[4], a.ints[9] * 4,
                                      ctx.stream);
  status(ctx, rc, rc == 3 ? "attention_kv4: work is too small" : "attention_kv4: q, kv and out must be 16-byte aligned, B at most 65535, P at most 2^27");
}

// kv4_reorder_gpu: kv u8[L, B, 2, kvh, 72 P], parents i64[B], n i64[1] (in place)
void runKv4Reorder(ExecCtx& ctx, const KernelArgs& a) {
  LK_REQUIRE(ctx, kv4Layout(a.ints[2], a.ints[4]) && a.ints[5] == a.ints[1] && a.ints[6] == 1 && a.ints[1] > 0 &&
                      a.ints[1] <= lkd::kMaxBeams && a.ints[3] > 0 && a.ints[0] * 2 * a.ints[3] <= 65535,
             "kv4_reorder: kv u8[L, B, 2, kvh, 72 P] with B <= 32 and L kvh <= 32767, parents i64[B], n i64[1]");
  status(ctx, lk_hip_kv4_reorder(a.ptrs[0], P<int64_t>(a, 1), P<int64_t>(a, 2), a.ints[0], a.ints[1],
                                 static_cast<int>(a.ints[3]), a.ints[4] / 72, ctx.stream),
         "kv4_reorder: launch failed");
}

}  // namespace

void registerKv4Kernels() {
  const Device G = Device::Gpu;
  registerKernel({"kv4_write_f16_gpu", G, runKv4Write, 4, 0});
  registerKernel({"qknorm_rope_kv4_f16_gpu", G, runKv4Qkr, 5, 1});
  registerKernel({"kv4_read_f16_gpu", G, runKv4Read, 1, 1});
  registerKernel({"attention_kv4_f16_gpu", G, runKv4Attention, 3, 2});
  registerKernel({"kv4_reorder_gpu", G, runKv4Reorder, 3, 0});
}

}  // namespace lkh
