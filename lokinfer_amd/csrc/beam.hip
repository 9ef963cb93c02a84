// Beam search's selection (lk.ops.beam_select_f32_gpu; no counterpart in the reference, which decodes greedily).
//
//   candidate (b, t) of an unfinished beam: score[b] + logits[b, t] - log sum_j exp(logits[b, j]);
//   of a finished one: score[b] at t = eos[0], nothing elsewhere.
// The k best of all B V: a beam's own by their logits, which candidates in 64 bits may not tell apart; equal logits to the lowest t,
// equal candidates of different beams to the lowest b. What has no value (a NaN, a row without a finite log-sum, a beam whose
// score is not finite) counts as -inf.
//
// Two launches. beamScanKernel passes once over the logits, 8192 of a row per workgroup, 32 per lane in registers, and leaves
// their k best, maximum and sum of exponentials. At least k of a wave's 64 lane maxima, so k of its logits, are not below the
// k-th largest of them (found by counting); the logits not below the largest such bound of the four waves, k and some
// more, go to LDS and are ranked by counting. Where they are more than fit (thousands of equal logits), each wave takes
// its k best one after the other instead. beamPickKernel, one workgroup, joins a row's lists with one wave (what is not
// below a bound from the lists' heads, ranked by counting), adds up its log-sum, and joins the rows' candidates likewise.
// Within a row the order is that of the logits (exact); between beams that of the candidates in 64 bits, the sums of
// exponentials of 8192 logits each (32 bits) added in 64 bits.
#include <algorithm>

#include "common.h"
#include "lokinfer_hip.h"

namespace lkd {

constexpr int kBeamMost = 32;    // beams and k
constexpr int kBeamWaves = 4;    // per workgroup of the scan
constexpr int kBeamTile = 8192;  // its logits, 32 per lane
constexpr int kBeamFit = 256;    // logits of a tile that are ranked by counting: one per thread, at least 4 kBeamMost
constexpr int kBeamLists = 32;   // lists per row at most: V <= 262144

struct BeamParams {
  const float* logits;   // [B, V]
  const float* scores;   // [B]
  const int64_t* done;   // [B]
  float2* sums;          // [B, tiles]: max, sum
  uint2* lists;          // [B, tiles, k]: (order of the logit, index), best first
  float* outScores;      // [k]
  int64_t* outParents;
  int64_t* outTokens;
  int64_t* outDone;
  int64_t v;
  int b, k, tiles;
  int eos[4];
};

// order-preserving key: larger logit, larger key; 0 is below all. NaN counts as -inf, -0 as 0
__device__ __forceinline__ unsigned orderOf(float x) {
  const unsigned u = __float_as_uint((x == x ? x : -INFINITY) + 0.0f);
  return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float valueOf(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

typedef unsigned long long u64;
__device__ __forceinline__ u64 pairOf(unsigned hi, unsigned lo) { return (static_cast<u64>(hi) << 32) | lo; }

// the wave's largest value, in every lane
template <int CTRL>
__device__ __forceinline__ unsigned maxDpp(unsigned v) {
  return max(v, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ unsigned waveMaxU32(unsigned v) {
  v = maxDpp<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v = maxDpp<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v = maxDpp<0x141>(v);  // row_half_mirror
  v = maxDpp<0x140>(v);  // row_mirror
  const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(p[0], p[1]);
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(h[0], h[1]);
}
__device__ __forceinline__ u64 waveMaxU64(unsigned hi, unsigned lo) {
  const unsigned top = waveMaxU32(hi);
  return pairOf(top, waveMaxU32(hi == top ? lo : 0u));
}

// how many of n keys come before the i-th, key: larger ones, and equal ones in front of it
__device__ __forceinline__ int beamRank(const u64* keys, int n, u64 key, int i) {
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < n; ++j) rank += keys[j] > key || (keys[j] == key && j < i);
  return rank;
}

// 151936 logits of 4 beams 6.1 us, of 16 beams, k = 16, 9.6 (9.7 MB): latency of one pass of loads, a reduction and the ranking.
__global__ __launch_bounds__(64 * kBeamWaves) void beamScanKernel(BeamParams p) {
  __shared__ u64 fit[kBeamFit];
  __shared__ unsigned bounds[kBeamWaves];
  __shared__ int count;
  __shared__ float2 part[kBeamWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tile = blockIdx.x, beam = blockIdx.y;
  const float* x = p.logits + static_cast<int64_t>(beam) * p.v;
  constexpr int E = kBeamTile / (64 * kBeamWaves);
  const unsigned first = static_cast<unsigned>(tile) * kBeamTile + wave * 64 * E + lane;
  unsigned key[E];
  float val[E], m = -INFINITY;
  const unsigned v = static_cast<unsigned>(p.v);
#pragma unroll
  for (int e = 0; e < E; ++e) val[e] = x[min(first + 64 * e, v - 1)];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool in = first + 64 * e < v;
    val[e] = in ? val[e] : -INFINITY;
    key[e] = in ? orderOf(val[e]) : 0u;
    m = fmaxf(m, val[e]);
  }
  m = waveMaxDpp(m);
  float s = 0.0f;
  const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((val[e] - base) * kLog2e);  // a NaN stays one; inf - inf is one
  s = waveSumDpp(s);
  if (lane == 0) part[wave] = make_float2(m, s);
  unsigned top = key[0];
#pragma unroll
  for (int e = 1; e < E; ++e) top = max(top, key[e]);
  int above = 0;
#pragma unroll
  for (int i = 0; i < 64; ++i) above += static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(top), i)) > top;
  // the smallest of the lane maxima with fewer than k above them
  const unsigned bound = ~waveMaxU32(above < p.k ? ~top : 0u);
  if (lane == 0) bounds[wave] = bound;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  unsigned least = bounds[0];
#pragma unroll
  for (int w = 1; w < kBeamWaves; ++w) least = max(least, bounds[w]);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (key[e] >= least) {
      const int at = atomicAdd(&count, 1);
      if (at < kBeamFit) fit[at] = pairOf(key[e], ~(first + 64 * e));
    }
  __syncthreads();
  int n = count;
  if (n > kBeamFit) {  // the same for every thread
    __syncthreads();
    for (int j = 0; j < p.k; ++j) {
      unsigned bk = key[0], be = 0u;  // equal keys of one lane: the first has the smallest index
#pragma unroll
      for (int e = 1; e < E; ++e) {
        const bool more = key[e] > bk;
        bk = more ? key[e] : bk;
        be = more ? e : be;
      }
      const u64 best = waveMaxU64(bk, ~(first + 64 * be));
      if (lane == 0) fit[wave * p.k + j] = best;
      const unsigned at = ~static_cast<unsigned>(best) - first;  // a multiple of 64 below 64 E in the lane that holds it
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at == 64u * e) key[e] = 0u;
    }
    __syncthreads();
    n = kBeamWaves * p.k;
  }
  if (static_cast<int>(threadIdx.x) < n) {  // (places without a logit can be equal: key 0)
    const u64 mine = fit[threadIdx.x];
    const int rank = beamRank(fit, n, mine, static_cast<int>(threadIdx.x));
    if (rank < p.k)
      p.lists[(static_cast<int64_t>(beam) * p.tiles + tile) * p.k + rank] =
          make_uint2(static_cast<unsigned>(mine >> 32), ~static_cast<unsigned>(mine));
  }
  if (threadIdx.x == 0) {
    float mm = -INFINITY, ss = 0.0f;
    for (int w = 0; w < kBeamWaves; ++w) mm = fmaxf(mm, part[w].x);
    for (int w = 0; w < kBeamWaves; ++w)
      ss += part[w].x == -INFINITY ? (part[w].y == part[w].y ? 0.0f : part[w].y) : part[w].y * expf(part[w].x - mm);
    p.sums[static_cast<int64_t>(beam) * p.tiles + tile] = make_float2(mm, ss);
  }
}

// the wave's own LDS, between its lanes' writes and reads
__device__ __forceinline__ void waveFence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Of `lists` lists of k keys each, best first, one wave keeps, in place and in order, those not below a bound that k of them
// reach, and returns their number. With d = ceil(k / lists) - 1, the J = ceil(k / (d + 1)) lists of the largest keys at
// place d have d + 1 keys each that are not below the smallest of these.
__device__ __forceinline__ int beamKeep(u64* keys, int lists, int k) {
  const int lane = threadIdx.x & 63, d = (k + lists - 1) / lists - 1, n = lists * k;
  waveFence();
  const u64 mine = lane < lists ? keys[lane * k + d] : 0;
  int above = 0;
#pragma unroll 4
  for (int i = 0; i < lists; ++i) above += keys[i * k + d] > mine;
  const u64 least = lane < lists && above * (d + 1) < k ? ~mine : 0;
  const u64 bound = ~waveMaxU64(static_cast<unsigned>(least >> 32), static_cast<unsigned>(least));
  int kept = 0;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const u64 key = i0 + lane < n ? keys[i0 + lane] : 0;
    const bool in = i0 + lane < n && key >= bound;
    const u64 all = __ballot(in);
    waveFence();  // places at or in front of those just read
    if (in) keys[kept + static_cast<int>(__popcll(all & ((u64{1} << lane) - 1)))] = key;
    kept += static_cast<int>(__popcll(all));
  }
  waveFence();
  return kept;
}

// an order-preserving key of a candidate; never 0
__device__ __forceinline__ u64 orderOf(double c) {
  const u64 u = static_cast<u64>(__double_as_longlong(c == 0.0 ? 0.0 : c));
  return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double valueOf(u64 key) {
  return __longlong_as_double(static_cast<long long>((key >> 63) ? key ^ 0x8000000000000000ull : ~key));
}

// Row `beam`'s k candidates, best first, by one wave: cand their keys (0: none left), tok their tokens.
__device__ __forceinline__ void beamRow(const BeamParams& p, int beam, u64* heads, u64* cand, int* tok) {
  const int lane = threadIdx.x & 63;
  const int64_t at = static_cast<int64_t>(beam) * p.tiles;
  const float score = p.scores[beam];
  const float2 mine = lane < p.tiles ? p.sums[at + lane] : make_float2(-INFINITY, 0.0f);
  const uint2* lists = p.lists + at * p.k;
  const int entries = p.tiles * p.k;
  waveFence();  // the row before
  for (int i0 = lane; i0 < entries; i0 += 64 * 8) {  // 8 loads in flight
    uint2 e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = lists[min(i0 + 64 * i, entries - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + 64 * i < entries) heads[i0 + 64 * i] = pairOf(e[i].x, ~e[i].y);
  }
  const float m = waveMaxDpp(mine.x);
  double sum = mine.x == -INFINITY ? (mine.y == mine.y ? 0.0 : mine.y)
                                   : mine.y * exp(static_cast<double>(mine.x) - static_cast<double>(m));
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const bool done = p.done[beam] != 0, live = fabsf(score) < INFINITY;
  if (done || !live || !(sum > 0.0 && fabsf(m) < INFINITY)) {
    // at most the finished beam's eos; else tokens in order, without a value
    const bool one = done && live;
    for (int j = lane; j < p.k; j += 64) {
      const int t = one ? (j == 0 ? p.eos[0] : j - 1 + (j - 1 >= p.eos[0])) : j;
      tok[j] = t;
      cand[j] = t < p.v ? orderOf(one && j == 0 ? static_cast<double>(score) : -INFINITY) : 0;
    }
    return;
  }
  const double lse = static_cast<double>(m) + log(sum);
  const int n = beamKeep(heads, p.tiles, p.k);
  for (int i = lane; i < n; i += 64) {
    const u64 key = heads[i];
    const int rank = beamRank(heads, n, key, i);
    if (rank >= p.k) continue;
    const unsigned order = static_cast<unsigned>(key >> 32);  // 0: fewer than k logits, none left
    const double c = static_cast<double>(score) + (static_cast<double>(valueOf(order)) - lse);
    cand[rank] = order == 0u ? 0 : orderOf(c == c ? c : -INFINITY);
    tok[rank] = static_cast<int>(~static_cast<unsigned>(key));
  }
}

// one workgroup: a wave per row (rows w, w + waves, ...), then a thread per candidate of the rows. B = k = 4 5.8 us, 16 12.6
// (k rounds of a wave's maximum for each of the two joins: 14.4): latency of LDS and of the two reductions in 64 bits.
__global__ __launch_bounds__(1024) void beamPickKernel(BeamParams p) {
  extern __shared__ u64 heads[];  // [waves, tiles, k]
  __shared__ u64 cand[kBeamMost * kBeamMost];
  __shared__ int tok[kBeamMost * kBeamMost];
  const int wave = threadIdx.x >> 6;
  for (int beam = wave; beam < p.b; beam += blockDim.x / 64)
    beamRow(p, beam, heads + static_cast<int64_t>(wave) * p.tiles * p.k, cand + beam * p.k, tok + beam * p.k);
  __syncthreads();
  for (int i = threadIdx.x; i < p.b * p.k; i += blockDim.x) {
    const u64 key = cand[i];
    const int beam = i / p.k;
    // in front of it: those of its own row, and of each other row from the best on what is larger or, of a lower beam, equal
    int rank = i - beam * p.k, l = beam == 0 ? 1 : 0, at = 0;
    while (rank < p.k && l < p.b) {
      const u64 other = at < p.k ? cand[l * p.k + at] : 0;
      const bool more = at < p.k && (other > key || (other == key && l < beam));
      rank += more;
      at = more ? at + 1 : 0;
      l = more ? l : l + 1 + (l + 1 == beam);
    }
    if (rank >= p.k) continue;  // at least k are candidates: k <= B V
    const int t = tok[i];
    p.outScores[rank] = static_cast<float>(valueOf(key));
    p.outParents[rank] = beam;
    p.outTokens[rank] = t;
    bool end = p.done[beam] != 0;
    for (int e = 0; e < 4; ++e) end = end || t == p.eos[e];
    p.outDone[rank] = end ? 1 : 0;
  }
}

}  // namespace lkd

namespace {

int64_t beamTiles(int64_t v) { return (v + lkd::kBeamTile - 1) / lkd::kBeamTile; }

}  // namespace

extern "C" {

int64_t lk_hip_beam_select_workspace_bytes(int64_t b, int64_t v, int k) {
  if (b <= 0 || v <= 0 || k <= 0) return 0;
  return (b * beamTiles(v) * (8 + 8 * static_cast<int64_t>(k)) + 15) / 16 * 16;
}

int lk_hip_beam_select_f32(const float* logits, const float* scores, const int64_t* done, float* out_scores,
                           int64_t* out_parents, int64_t* out_tokens, int64_t* out_done, int64_t b, int64_t v, int k,
                           const int* eos, int num_eos, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lkd;
  if (b <= 0 || b > kBeamMost || k <= 0 || k > kBeamMost || v <= 0 || v > int64_t{kBeamTile} * kBeamLists || k > b * v ||
      num_eos < 1 || num_eos > 4)
    return 1;
  for (int i = 0; i < num_eos; ++i)
    if (eos[i] < 0 || eos[i] >= v) return 1;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < lk_hip_beam_select_workspace_bytes(b, v, k))
    return 3;
  BeamParams p{};
  p.logits = logits;
  p.scores = scores;
  p.done = done;
  p.tiles = static_cast<int>(beamTiles(v));
  p.lists = static_cast<uint2*>(workspace);
  p.sums = reinterpret_cast<float2*>(static_cast<char*>(workspace) + b * p.tiles * k * 8);
  p.outScores = out_scores;
  p.outParents = out_parents;
  p.outTokens = out_tokens;
  p.outDone = out_done;
  p.v = v;
  p.b = static_cast<int>(b);
  p.k = k;
  for (int i = 0; i < 4; ++i) p.eos[i] = i < num_eos ? eos[i] : -1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(beamScanKernel, dim3(static_cast<unsigned>(p.tiles), static_cast<unsigned>(b)),
                     dim3(64 * kBeamWaves), 0, s, p);
  // as many rows at a time as their lists fit 48 KiB (one row's: at most 16)
  const int64_t row = int64_t{8} * p.tiles * k;
  const int waves = static_cast<int>(std::min<int64_t>({b, 16, (48 << 10) / row}));
  hipLaunchKernelGGL(beamPickKernel, dim3(1), dim3(static_cast<unsigned>(64 * waves)), static_cast<size_t>(waves * row), s, p);
  return hipGetLastError() == hipSuccess ? 0 : 2;
}

}  // extern "C"

namespace lkh {

namespace {

// beam_select_f32_gpu: logits[B, V], scores[B], done i64[B] -> scores f32[k], parents, tokens, done i64[k], work f32[n];
// attr eos (1 .. 4 ints)
void runBeamSelect(ExecCtx& ctx, const KernelArgs& a) {
  const int64_t b = a.ints[0], v = a.ints[1], k = a.ints[4];
  LK_REQUIRE(ctx, a.ints[2] == b && a.ints[3] == b && a.ints[5] == k && a.ints[6] == k && a.ints[7] == k && k > 0 &&
                      k <= lkd::kBeamMost && a.numInts >= 10 && a.numInts <= 13,
             "beam_select: logits f32[B, V], scores f32[B], done i64[B], k outputs, 1 to 4 eos ids");
  int eos[4];
  const int num = static_cast<int>(a.numInts) - 9;
  for (int i = 0; i < num; ++i) {
    LK_REQUIRE(ctx, a.ints[9 + i] >= 0 && a.ints[9 + i] < v, "beam_select: an eos id is out of range");
    eos[i] = static_cast<int>(a.ints[9 + i]);
  }
  const int rc = lk_hip_beam_select_f32(P<float>(a, 0), P<float>(a, 1), P<int64_t>(a, 2), P<float>(a, 3), P<int64_t>(a, 4),
                                        P<int64_t>(a, 5), P<int64_t>(a, 6), b, v, static_cast<int>(k), eos, num, a.ptrs[7],
                                        a.ints[8] * 4, ctx.stream);
  status(ctx, rc, rc == 3 ? "beam_select: work is too small" : "beam_select: at most 32 beams, k <= 32, V <= 262144");
}

}  // namespace

void registerBeamKernels() { registerKernel({"beam_select_f32_gpu", Device::Gpu, runBeamSelect, 3, 5}); }

}  // namespace lkh
