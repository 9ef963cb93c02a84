// Key / value caches held in 4 bits (lk.ops.q4_gpu; no counterpart in the reference, whose caches are f16 or f32).
//
// A cache is u8 [B, 2, kvh, 72 P] (B sequences; keys, values; P rows, a multiple of 32): per (sequence, key or value, kv
// head) P rows of 64 bytes of codes, then P rows of 4 f16 scales, one for each 32 of the head's 128 values (format: q4.h).
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
// One wave quantises a row's key (lanes 0..31) and value (lanes 32..63), 4 values per lane: x of the lane's
// values 4 (lane % 32) ... kvBlock: the (sequence, kv head)'s key block; its value block lies valueOff bytes further.
__device__ __forceinline__ void kv4PutRow(half4 x, char* kvBlock, int64_t valueOff, int64_t cap, int64_t row) {
  const int lane = threadIdx.x & 63, l = lane & 31;
  float v[4], hi = 0.0f, lo = 0.0f;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = static_cast<float>(x[e]);
    hi = fmaxf(hi, v[e]);
    lo = fminf(lo, v[e]);
    bad = bad || !(fabsf(v[e]) < INFINITY);
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {  // the 8 lanes of a group
    hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    lo = fminf(lo, __shfl_xor(lo, o, 64));
  }
  const bool rowBad = __any(bad);
  float s = q4Scale(hi, lo);
  if (rowBad) s = lane < 32 ? __builtin_nanf("") : 0.0f;
  unsigned word = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) word |= q4Code(v[e], s) << q4Shift(4 * (l & 1) + e);
  word |= __shfl_xor(word, 1, 64);
  char* at = kvBlock + (lane < 32 ? 0 : valueOff);
  if ((l & 1) == 0) *reinterpret_cast<unsigned*>(at + row * 64 + 2 * l) = word;
  if ((l & 7) == 0) *reinterpret_cast<h16*>(at + cap * 64 + row * 8 + l / 4) = static_cast<h16>(s);
}

__global__ __launch_bounds__(256) void kv4WriteKernel(char* __restrict__ kv, const h16* __restrict__ k,
                                                      const h16* __restrict__ v, const int64_t* __restrict__ pos,
                                                      int64_t b, int64_t t, int kvh, int64_t cap) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (item >= b * t * kvh) return;
  const int64_t seqRow = item / kvh, seq = seqRow / t, row = pos[seq] + (seqRow - seq * t);
  const int h = static_cast<int>(item - seqRow * kvh);
  if (row < 0 || row >= cap) return;  // uniform over the wave
  const h16* src = (lane < 32 ? k : v) + seqRow * kvh * KHD + h * KHD + 4 * (lane & 31);
  const int64_t block = 72 * cap;
  kv4PutRow(*reinterpret_cast<const half4*>(src), kv + (seq * 2 * kvh + h) * block, kvh * block, cap, row);
}

struct Kv4QkrParams {
  const h16* qkv;
  const h16* qg;
  const h16* kg;
  const int64_t* pos;
  char* kv;
  h16* q;
  int64_t b, t, cap;
  int qh, kvh;
  float eps;
  RopeTable tab;
};

// One wave per (row, q head) and (row, kv head): a q head is normalized and rotated to q, a kv head's key likewise and
// quantised with its value. Arithmetic and roundings of the norm and the rotation as qkRopeKvKernel's.
__global__ __launch_bounds__(256) void kv4QkRopeKernel(Kv4QkrParams p) {
  __shared__ __attribute__((aligned(16))) h16 rows[4][2 * KHD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slots = p.qh + p.kvh;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  if (item >= p.b * p.t * slots) return;
  const int64_t r = item / slots, seq = r / p.t, row = p.pos[seq] + (r - seq * p.t);
  const int slot = static_cast<int>(item - r * slots);
  const int64_t width = static_cast<int64_t>(p.qh + 2 * p.kvh) * KHD;
  const bool isQ = slot < p.qh;
  if (!isQ && (row < 0 || row >= p.cap)) return;
  const h16* x = p.qkv + r * width + slot * KHD;
  const h16* g = isQ ? p.qg : p.kg;
  const float f = rmsFactor(rowSumSq(x, KHD, lane), KHD, p.eps);
  h16 a, b;
  ropePair(static_cast<float>(rmsElem(x[lane], g[lane], f)), static_cast<float>(rmsElem(x[lane + 64], g[lane + 64], f)),
           row, p.tab.invf[lane], a, b);
  if (isQ) {
    h16* o = p.q + r * p.qh * KHD + slot * KHD;
    o[lane] = a;
    o[lane + 64] = b;
    return;
  }
  const h16* v = x + static_cast<int64_t>(p.kvh) * KHD;
  h16* mine = rows[wave];
  mine[lane] = a;
  mine[lane + 64] = b;
  mine[KHD + lane] = v[lane];
  mine[KHD + lane + 64] = v[lane + 64];
  // this wave's own slice: its LDS operations complete in order
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const int64_t block = 72 * p.cap;
  kv4PutRow(*reinterpret_cast<const half4*>(mine + 4 * lane), p.kv + (seq * 2 * p.kvh + (slot - p.qh)) * block,
            p.kvh * block, p.cap, row);
}

// ---- reading ----------------------------------------------------------------------------------------------------
// one thread per 8 values: blocks of 72 cap bytes -> f16 [blocks, cap, 128]
__global__ __launch_bounds__(256) void kv4ReadKernel(const char* __restrict__ kv, h16* __restrict__ out, int64_t blocks,
                                                     int64_t cap) {
  const int64_t total = blocks * cap * 16;
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < total;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = id >> 4, blk = r / cap, row = r - blk * cap;
    const int w = static_cast<int>(id & 15);
    const char* at = kv + blk * 72 * cap;
    const half8 v = q4Ints(*reinterpret_cast<const unsigned*>(at + row * 64 + 4 * w));
    const h16 s = *reinterpret_cast<const h16*>(at + cap * 64 + row * 8 + 2 * (w >> 2));
    half8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = v[e] * s;
    st8(out + 8 * id, y);
  }
}

// ---- attention ----------------------------------------------------------------------------------------------------
struct Kv4Params {
  const h16* q;  // [B T, qh 128]
  const char* kv;
  const int64_t* pos;
  h16* out;
  float* part;  // [splits, B T qh, 130]: (max, sum, out[128]) of each key range
  int64_t b, t, cap;
  int qh, kvh, splits;
  float scale;  // log2(e) / sqrt(128)
  unsigned long long* err;
};

// Rows of a kv head: r = i group + h, query i's q heads side by side; R of them per wave. Lane (key = lane / 4, g = lane % 4)
// holds the 32 dims of scale group g: a load instruction reads 16 whole rows. Keys 16 u + lane / 4 of the wave's 64-key
// chunks are one lane quad's own: it keeps their running max, sum and weighted values by itself, joined at the end.
template <int R>
__global__ __launch_bounds__(64) void kv4ChunkKernel(Kv4Params p) {
  __shared__ float red[R][64][33];
  const int lane = threadIdx.x, g = lane & 3, kl = lane >> 2;
  const int group = p.qh / p.kvh;
  const int64_t rowsHead = p.t * group, blocksHead = (rowsHead + R - 1) / R;
  int64_t id = blockIdx.x;
  const int64_t rb = id % blocksHead;
  id /= blocksHead;
  const int kvHead = static_cast<int>(id % p.kvh);
  const int64_t seq = id / p.kvh;
  const int split = blockIdx.y;
  const int64_t p0 = p.pos[seq];
  const bool bad = p0 < 0 || p0 + p.t > p.cap;
  int64_t nkRow[R];
  int64_t nk = 0;
  float qf[R][32];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = min<int64_t>(rb * R + r, rowsHead - 1), i = row / group, h = kvHead * group + (row - i * group);
    nkRow[r] = p0 < 0 ? 0 : min<int64_t>(p0 + i + 1, p.cap);
    nk = max(nk, nkRow[r]);
    const h16* q = p.q + (seq * p.t + i) * p.qh * KHD + h * KHD + 32 * g;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const half8 v = ld8(q + 8 * c);
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[r][8 * c + e] = static_cast<float>(v[e]);
    }
  }
  if (bad && split == 0 && rb == 0 && kvHead == 0 && lane == 0) raiseDeviceError(p.err, LK_DEVERR_POSITION, p0 < 0 ? p0 : p0 + p.t - 1);
  const int64_t chunks = (nk + 63) / 64, per = (chunks + p.splits - 1) / p.splits;
  const int64_t c0 = split * per, c1 = min(c0 + per, chunks);
  const int64_t block = 72 * p.cap;
  const char* kb = p.kv + (seq * 2 * p.kvh + kvHead) * block;
  const char* vb = kb + p.kvh * block;
  float m[R], l[R], acc[R][32];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int d = 0; d < 32; ++d) acc[r][d] = 0.0f;
  }
  for (int64_t c = c0; c < c1; ++c) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t key = c * 64 + 16 * u + kl, at = min(key, nk - 1);
      const uint4 kw = *reinterpret_cast<const uint4*>(kb + at * 64 + 16 * g);
      const uint4 vw = *reinterpret_cast<const uint4*>(vb + at * 64 + 16 * g);
      const float ks = static_cast<float>(*reinterpret_cast<const h16*>(kb + p.cap * 64 + at * 8 + 2 * g));
      const float vs = static_cast<float>(*reinterpret_cast<const h16*>(vb + p.cap * 64 + at * 8 + 2 * g));
      const unsigned kws[4] = {kw.x, kw.y, kw.z, kw.w}, vws[4] = {vw.x, vw.y, vw.z, vw.w};
      float dot[R];
#pragma unroll
      for (int r = 0; r < R; ++r) dot[r] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const half8 x = q4Ints(kws[w]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e) dot[r] = fmaf(static_cast<float>(x[e]), qf[r][8 * w + e], dot[r]);
      }
      float wgt[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float d = dot[r] * ks;
        d += __shfl_xor(d, 1, 64);
        d += __shfl_xor(d, 2, 64);
        const float s = key < nkRow[r] ? d * p.scale : -INFINITY;
        const float mx = fmaxf(m[r], s);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float corr = __builtin_amdgcn_exp2f(m[r] - base);
        const float e = __builtin_amdgcn_exp2f(s - base);
        l[r] = l[r] * corr + e;
        m[r] = mx;
        wgt[r] = e * vs;
        if (__any(corr != 1.0f)) {
#pragma unroll
          for (int d2 = 0; d2 < 32; ++d2) acc[r][d2] *= corr;
        }
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const half8 x = q4Ints(vws[w]);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[r][8 * w + e] = fmaf(static_cast<float>(x[e]), wgt[r], acc[r][8 * w + e]);
      }
    }
  }
  // join the 16 lane quads
  float mAll[R], lAll[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float mm = m[r];
#pragma unroll
    for (int o = 4; o < 64; o <<= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
    mAll[r] = mm;
    const float f = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - mm);
    float ll = m[r] == -INFINITY ? l[r] : l[r] * f;  // a NaN score leaves m alone: the NaN is in l
#pragma unroll
    for (int o = 4; o < 64; o <<= 1) ll += __shfl_xor(ll, o, 64);
    lAll[r] = ll;
#pragma unroll
    for (int d = 0; d < 32; ++d) red[r][lane][d] = acc[r][d] * f;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = rb * R + r;
    if (row >= rowsHead) continue;
    const int64_t i = row / group, h = kvHead * group + (row - i * group), at = (seq * p.t + i) * p.qh + h;
#pragma unroll
    for (int d0 = 0; d0 < KHD; d0 += 64) {
      const int d = d0 + lane;
      float o = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; ++j) o += red[r][4 * j + (d >> 5)][d & 31];
      if (p.splits == 1) {
        const bool noRow = p0 < 0 || p0 + i >= p.cap;
        p.out[at * KHD + d] = noRow ? static_cast<h16>(__builtin_nanf("")) : toH16(o / lAll[r]);
      } else {
        p.part[(split * p.b * p.t * p.qh + at) * (KHD + 2) + 2 + d] = o;
      }
    }
    if (p.splits > 1 && lane == 0) {
      float* pp = p.part + (split * p.b * p.t * p.qh + at) * (KHD + 2);
      pp[0] = mAll[r];
      pp[1] = lAll[r];
    }
  }
}

// one workgroup per (query, q head)
__global__ __launch_bounds__(128) void kv4MergeKernel(Kv4Params p) {
  const int d = threadIdx.x;
  const int64_t at = blockIdx.x, rows = p.b * p.t * p.qh, qi = at / p.qh, seq = qi / p.t, p0 = p.pos[seq] + (qi - seq * p.t);
  const bool noRow = p.pos[seq] < 0 || p0 >= p.cap;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part[(s * rows + at) * (KHD + 2)]);
  float l = 0.0f, o = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    const float* pp = p.part + (s * rows + at) * (KHD + 2);
    const float f = pp[0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pp[0] - m);  // no key: zeros, or a NaN to pass on
    l = fmaf(f, pp[1], l);
    o = fmaf(f, pp[2 + d], o);
  }
  p.out[at * KHD + d] = noRow ? static_cast<h16>(__builtin_nanf("")) : toH16(o / l);
}

// ---- moving caches between sequences ------------------------------------------------------------------------------
// One thread per 8 bytes of a (layer, key or value, kv head)'s live rows: it reads the piece of every sequence whose parent
// is another from that parent, then writes them, so that no write comes before a read of the same bytes.
constexpr int kMaxBeams = 32;
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
  for (int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; id < rows * 9;
       id += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t off = id < rows * 8 ? id * 8 : cap * 64 + (id - rows * 8) * 8;
    unsigned long long v[kMaxBeams];
#pragma unroll
    for (int i = 0; i < kMaxBeams; ++i)
      if (i < b) {
        const int64_t from = parents[i];
        v[i] = from >= 0 && from < b ? *reinterpret_cast<const unsigned long long*>(base + from * seqStride + off)
                                     : 0x7E007E007E007E00ull;  // NaN where it lands in the scales
      }
#pragma unroll
    for (int i = 0; i < kMaxBeams; ++i)
      if (i < b && parents[i] != i) *reinterpret_cast<unsigned long long*>(base + i * seqStride + off) = v[i];
  }
}

}  // namespace lkd

namespace {

bool al16(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; }
bool al8(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 7) == 0; }
int launched() { return hipGetLastError() == hipSuccess ? 0 : 2; }
bool kvOk(const void* kv, int64_t b, int kvh, int64_t cap) {
  return b > 0 && kvh > 0 && cap > 0 && cap % 32 == 0 && al16(kv);
}

}  // namespace

extern "C" {

int lk_hip_kv4_write(void* kv, const void* k, const void* v, const int64_t* pos, int64_t b, int64_t t, int kvh, int64_t cap,
                     void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || t < 0 || !al8(k) || !al8(v)) return 1;
  const int64_t items = b * t * kvh;
  if (items == 0) return 0;
  if (items > int64_t{4} * 0x7FFFFFFF) return 1;
  hipLaunchKernelGGL(kv4WriteKernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<char*>(kv), static_cast<const h16*>(k),
                     static_cast<const h16*>(v), pos, b, t, kvh, cap);
  return launched();
}

int lk_hip_kv4_qknorm_rope(const void* qkv, const void* qg, const void* kg, const int64_t* pos, void* kv, void* q, int64_t b,
                           int64_t t, int qh, int kvh, int64_t cap, float eps, float theta, void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || t < 0 || qh <= 0 || !al16(qkv)) return 1;
  const int64_t items = b * t * (qh + kvh);
  if (items == 0) return 0;
  if (items > int64_t{4} * 0x7FFFFFFF) return 1;
  Kv4QkrParams p{static_cast<const h16*>(qkv), static_cast<const h16*>(qg), static_cast<const h16*>(kg), pos,
                 static_cast<char*>(kv), static_cast<h16*>(q), b, t, cap, qh, kvh, eps, {}};
  for (int j = 0; j < 64; ++j) p.tab.invf[j] = 1.0f / std::pow(theta, static_cast<float>(2 * j) / 128.0f);
  hipLaunchKernelGGL(kv4QkRopeKernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return launched();
}

int lk_hip_kv4_read(const void* kv, void* out, int64_t blocks, int64_t cap, void* stream) {
  using namespace lkd;
  if (blocks < 0 || cap <= 0 || cap % 32 != 0 || !al16(kv) || !al16(out)) return 1;
  if (blocks == 0) return 0;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((blocks * cap * 16 + 255) / 256, 65536));
  hipLaunchKernelGGL(kv4ReadKernel, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const char*>(kv),
                     static_cast<h16*>(out), blocks, cap);
  return launched();
}

static int kv4Splits(int64_t b, int64_t t, int qh, int kvh, int64_t cap) {
  if (b <= 0 || t <= 0 || qh <= 0 || kvh <= 0 || qh % kvh != 0 || cap <= 0) return 1;
  const int64_t waves = b * kvh * ((t * (qh / kvh) + 1) / 2);
  const int64_t most = std::max<int64_t>(1, (cap + 63) / 64);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({most, 128, 2048 / std::max<int64_t>(waves, 1)})));
}

int64_t lk_hip_kv4_attention_workspace_bytes(int64_t b, int64_t t, int qh, int kvh, int64_t cap) {
  const int64_t s = kv4Splits(b, t, qh, kvh, cap);
  return s > 1 ? s * b * t * qh * (lkd::KHD + 2) * 4 : 0;
}

int lk_hip_kv4_attention(const void* q, const void* kv, const int64_t* pos, void* out, int64_t b, int64_t t, int qh, int kvh,
                         int64_t cap, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || t < 0 || qh <= 0 || qh % kvh != 0 || !al16(q)) return 1;
  if (t == 0) return 0;
  const int splits = kv4Splits(b, t, qh, kvh, cap);
  if (workspace_bytes < lk_hip_kv4_attention_workspace_bytes(b, t, qh, kvh, cap) || (splits > 1 && !workspace)) return 3;
  const Kv4Params p{static_cast<const h16*>(q), static_cast<const char*>(kv), pos, static_cast<h16*>(out),
                    static_cast<float*>(workspace), b, t, cap, qh, kvh, splits,
                    kLog2e / std::sqrt(static_cast<float>(KHD)), lkh::deviceErrorRecord()};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t blocks = b * kvh * ((t * (qh / kvh) + 1) / 2);
  if (blocks > 0x7FFFFFFF || b * t * qh > 0x7FFFFFFF) return 1;
  hipLaunchKernelGGL(kv4ChunkKernel<2>, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(splits)), dim3(64), 0, s, p);
  if (splits > 1)
    hipLaunchKernelGGL(kv4MergeKernel, dim3(static_cast<unsigned>(b * t * qh)), dim3(128), 0, s, p);
  return launched();
}

int lk_hip_kv4_reorder(void* kv, const int64_t* parents, const int64_t* n, int64_t layers, int64_t b, int kvh, int64_t cap,
                       void* stream) {
  using namespace lkd;
  if (!kvOk(kv, b, kvh, cap) || layers < 0 || b > kMaxBeams || layers * 2 * kvh > 65535) return 1;
  if (layers == 0) return 0;
  const unsigned gx = static_cast<unsigned>(std::min<int64_t>((cap * 9 + 255) / 256, 64));
  hipLaunchKernelGGL(kv4ReorderKernel, dim3(gx, static_cast<unsigned>(layers * 2 * kvh)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<char*>(kv), parents, n, layers, static_cast<int>(b), kvh,
                     cap, lkh::deviceErrorRecord());
  return launched();
}

}  // extern "C"

// ---- registry -----------------------------------------------------------------------------------------------------
namespace lkh {

namespace {

bool kv4Shape(int64_t two, int64_t bytes) { return two == 2 && bytes > 0 && bytes % (72 * 32) == 0; }

// kv4_write_f16_gpu: kv u8[B, 2, kvh, 72 P], k, v f16[B T, kvh 128], pos i64[B] (in place)
void runKv4Write(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t b = a.ints[0], kvh = a.ints[2], cap = a.ints[3] / 72, rows = a.ints[4];
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Shape(a.ints[1], a.ints[3]) && rows % b == 0 && a.ints[5] == kvh * 128 &&
                      a.ints[6] == rows && a.ints[7] == a.ints[5] && a.ints[8] == b,
             "kv4_write: kv u8[B, 2, kvh, 72 P] with P % 32 == 0, k and v f16[B T, kvh 128], pos i64[B]");
  status(ctx, lk_hip_kv4_write(a.ptrs[0], a.ptrs[1], a.ptrs[2], P<int64_t>(a, 3), b, rows / b, static_cast<int>(kvh), cap,
                               ctx.stream),
         "kv4_write: kv must be 16-byte, k and v 8-byte aligned");
}

// qknorm_rope_kv4_f16_gpu: qkv f16[B T, (qh + 2 kvh) 128], qg, kg f16[128], pos i64[B], kv (in place) -> q f16[B T, qh 128];
// floats eps, theta
void runKv4Qkr(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t rows = a.ints[0], b = a.ints[4], kvh = a.ints[7], cap = a.ints[8] / 72, qw = a.ints[10];
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Shape(a.ints[6], a.ints[8]) && a.ints[5] == b && rows % b == 0 &&
                      a.ints[2] == 128 && a.ints[3] == 128 && qw > 0 && qw % 128 == 0 &&
                      a.ints[1] == qw + 2 * kvh * 128 && a.ints[9] == rows,
             "qknorm_rope_kv4: qkv f16[B T, (qh + 2 kvh) 128], gains f16[128], pos i64[B], kv u8[B, 2, kvh, 72 P]");
  status(ctx, lk_hip_kv4_qknorm_rope(a.ptrs[0], a.ptrs[1], a.ptrs[2], P<int64_t>(a, 3), a.ptrs[4], a.ptrs[5], b, rows / b,
                                     static_cast<int>(qw / 128), static_cast<int>(kvh), cap, F(a, 0, 1e-6f), F(a, 1, 1e6f),
                                     ctx.stream),
         "qknorm_rope_kv4: qkv and kv must be 16-byte aligned");
}

// kv4_read_f16_gpu: kv u8[blocks, 72 P] -> f16[blocks, P, 128]
void runKv4Read(ExecCtx& ctx, const KernelArgs& a) {
  LK_REQUIRE(ctx, kv4Shape(2, a.ints[1]) && a.ints[2] == a.ints[0] && a.ints[3] == a.ints[1] / 72 && a.ints[4] == 128,
             "kv4_read: kv u8[blocks, 72 P] with P % 32 == 0, out f16[blocks, P, 128]");
  status(ctx, lk_hip_kv4_read(a.ptrs[0], a.ptrs[1], a.ints[0], a.ints[3], ctx.stream), "kv4_read: launch failed");
}

// attention_kv4_f16_gpu: q f16[B T, qh 128], kv u8[B, 2, kvh, 72 P], pos i64[B] -> out f16[B T, qh 128], work f32[n]
void runKv4Attention(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t rows = a.ints[0], width = a.ints[1], b = a.ints[2], kvh = a.ints[4], cap = a.ints[5] / 72;
  LK_REQUIRE(ctx, b > 0 && kvh > 0 && kv4Shape(a.ints[3], a.ints[5]) && rows % b == 0 && width > 0 &&
                      width % (128 * kvh) == 0 && a.ints[6] == b && a.ints[7] == rows && a.ints[8] == width,
             "attention_kv4: q f16[B T, qh 128], kv u8[B, 2, kvh, 72 P], qh a multiple of kvh, pos i64[B]");
  const int rc = lk_hip_kv4_attention(a.ptrs[0], a.ptrs[1], P<int64_t>(a, 2), a.ptrs[3], b, rows / b,
                                      static_cast<int>(width / 128), static_cast<int>(kvh), cap, a.ptrs[4], a.ints[9] * 4,
                                      ctx.stream);
  status(ctx, rc, rc == 3 ? "attention_kv4: work is too small" : "attention_kv4: q and kv must be 16-byte aligned");
}

// kv4_reorder_gpu: kv u8[L, B, 2, kvh, 72 P], parents i64[B], n i64[1] (in place)
void runKv4Reorder(ExecCtx& ctx, const KernelArgs& a) {
  LK_REQUIRE(ctx, kv4Shape(a.ints[2], a.ints[4]) && a.ints[5] == a.ints[1] && a.ints[6] == 1 && a.ints[1] > 0 &&
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
