// Beam search's selection (lk.ops.beam_select_f32_gpu; no counterpart in the reference, which decodes greedily).
//
//   candidate (b, t) of an unfinished beam: score[b] + logits[b, t] - log sum_j exp(logits[b, j]);
//   of a finished one: score[b] at t = eos[0], nothing elsewhere.
// The k best of all B V, ties to the lowest b V + t. What has no value (a NaN, a row without a finite log-sum, a beam whose
// score is not finite) counts as -inf.
//
// Three launches: beamScanKernel, one pass over the logits: each wave takes 1024 of a row, keeps them in registers, and
// leaves their maximum, sum of exponentials and k best; beamRowKernel joins a row's; beamPickKernel takes the k best
// of the beams' lists. Within a row the order is that of the logits (exact); between beams that of the candidates in
// 64 bits, the sum of exponentials added in 64 bits over the waves' 32-bit sums.
#include <algorithm>

#include "common.h"
#include "lokinfer_hip.h"

namespace lkd {

constexpr int kBeamMost = 32;    // beams and k
constexpr int kBeamWave = 1024;  // logits per wave
constexpr int kBeamLists = 256;  // waves per row

struct BeamParams {
  const float* logits;   // [B, V]
  const float* scores;   // [B]
  const int64_t* done;   // [B]
  float* sums;           // [B, waves, 2]: max, sum
  uint2* lists;          // [B, waves, k]: (order of the logit, index), best first
  double* cand;          // [B, k]
  int* tok;              // [B, k]
  float* outScores;      // [k]
  int64_t* outParents;
  int64_t* outTokens;
  int64_t* outDone;
  int64_t v;
  int b, k, waves;
  int eos[4];
};

// order-preserving key: larger logit, larger key; 0 is below all. NaN counts as -inf, -0 as 0
__device__ __forceinline__ unsigned orderOf(float x) {
  if (!(x == x)) x = -INFINITY;
  const unsigned u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float valueOf(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

// the wave's best (key, index): the larger key, then the smaller index
__device__ __forceinline__ void waveBest(unsigned& key, unsigned& idx) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned k2 = __shfl_xor(key, o, 64), i2 = __shfl_xor(idx, o, 64);
    if (k2 > key || (k2 == key && i2 < idx)) {
      key = k2;
      idx = i2;
    }
  }
}

__global__ __launch_bounds__(256) void beamScanKernel(BeamParams p) {
  const int lane = threadIdx.x & 63, w = blockIdx.x * 4 + (threadIdx.x >> 6), beam = blockIdx.y;
  if (w >= p.waves) return;
  const float* x = p.logits + static_cast<int64_t>(beam) * p.v;
  const int64_t first = static_cast<int64_t>(w) * kBeamWave;
  constexpr int E = kBeamWave / 64;
  unsigned key[E];
  float m = -INFINITY;
  float val[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t i = first + lane + 64 * e;
    val[e] = i < p.v ? x[i] : -INFINITY;
    key[e] = i < p.v ? orderOf(val[e]) : 0u;
    m = fmaxf(m, val[e]);
  }
  m = waveMax(m);
  float s = 0.0f;
  const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int e = 0; e < E; ++e) s += expf(val[e] - base);  // a NaN stays one; inf - inf is one
  s = waveSum(s);
  const int64_t at = static_cast<int64_t>(beam) * p.waves + w;
  if (lane == 0) {
    p.sums[2 * at] = m;
    p.sums[2 * at + 1] = s;
  }
  for (int j = 0; j < p.k; ++j) {
    unsigned bk = 0u, be = 0u;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] > bk) {
        bk = key[e];
        be = e;
      }
    unsigned wk = bk, wi = lane + 64 * be;  // equal keys of one lane: the first, its smallest index
    waveBest(wk, wi);
    if (lane == 0) p.lists[at * p.k + j] = make_uint2(wk, static_cast<unsigned>(first) + wi);
    if ((wi & 63) == static_cast<unsigned>(lane)) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (static_cast<unsigned>(e) == wi >> 6) key[e] = 0u;
    }
  }
}

// one wave per beam: the row's log-sum, then k times the best head of its lists
__global__ __launch_bounds__(64) void beamRowKernel(BeamParams p) {
  extern __shared__ uint2 heads[];  // [waves, k]
  const int lane = threadIdx.x, beam = blockIdx.x;
  const int64_t at = static_cast<int64_t>(beam) * p.waves;
  double* cand = p.cand + static_cast<int64_t>(beam) * p.k;
  int* tok = p.tok + static_cast<int64_t>(beam) * p.k;
  const float score = p.scores[beam];
  float m = -INFINITY;
  for (int w = lane; w < p.waves; w += 64) m = fmaxf(m, p.sums[2 * (at + w)]);
  m = waveMax(m);
  double sum = 0.0;
  for (int w = lane; w < p.waves; w += 64) {
    const float mw = p.sums[2 * (at + w)];
    const double part = static_cast<double>(p.sums[2 * (at + w) + 1]);
    sum += mw == -INFINITY ? (part == part ? 0.0 : part) : part * exp(static_cast<double>(mw) - static_cast<double>(m));
  }
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const bool done = p.done[beam] != 0;
  const bool live = fabsf(score) < INFINITY;
  if (done || !live || !(sum > 0.0 && fabsf(m) < INFINITY)) {
    // at most the finished beam's eos; else tokens in order, without a value
    const bool one = done && live;
    for (int j = lane; j < p.k; j += 64) {
      const int t = one ? (j == 0 ? p.eos[0] : j - 1 + (j - 1 >= p.eos[0])) : j;
      tok[j] = t < p.v ? t : -1;
      cand[j] = one && j == 0 ? static_cast<double>(score) : -INFINITY;
    }
    return;
  }
  const double lse = static_cast<double>(m) + log(sum);
  for (int i = lane; i < p.waves * p.k; i += 64) heads[i] = p.lists[at * p.k + i];
  constexpr int L = kBeamLists / 64;
  int next[L];
#pragma unroll
  for (int i = 0; i < L; ++i) next[i] = 0;
  __syncthreads();
  for (int j = 0; j < p.k; ++j) {
    unsigned bk = 0u, bi = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int w = lane + 64 * i;
      if (w < p.waves && next[i] < p.k) {
        const uint2 h = heads[w * p.k + next[i]];
        if (h.x > bk || (h.x == bk && h.x != 0u && h.y < bi)) {
          bk = h.x;
          bi = h.y;
        }
      }
    }
    waveBest(bk, bi);
    const bool any = bk != 0u;  // fewer than k logits: none left
    if (lane == 0) {
      const double c = any ? static_cast<double>(score) + (static_cast<double>(valueOf(bk)) - lse) : -INFINITY;
      cand[j] = c == c ? c : -INFINITY;
      tok[j] = any ? static_cast<int>(bi) : -1;
    }
    const int w = static_cast<int>(bi / kBeamWave);
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (any && w == lane + 64 * i) ++next[i];
  }
}

// one wave: k times the best head of the beams' lists; lane b holds beam b's
__global__ __launch_bounds__(64) void beamPickKernel(BeamParams p) {
  const int lane = threadIdx.x;
  int next = 0;
  for (int j = 0; j < p.k; ++j) {
    // a list that is used up, or a token that is not there, is below every -inf
    double c = -INFINITY;
    int t = -1;
    if (lane < p.b && next < p.k) {
      c = p.cand[lane * p.k + next];
      t = p.tok[lane * p.k + next];
    }
    int who = lane;
    bool has = t >= 0;
    for (int o = 32; o > 0; o >>= 1) {
      const double c2 = __shfl_xor(c, o, 64);
      const int w2 = __shfl_xor(who, o, 64), t2 = __shfl_xor(t, o, 64), h2 = __shfl_xor(static_cast<int>(has), o, 64);
      const bool other = h2 && (!has || c2 > c || (c2 == c && w2 < who));
      if (other) {
        c = c2;
        who = w2;
        t = t2;
        has = true;
      }
    }
    if (lane == 0) {
      p.outScores[j] = static_cast<float>(c);
      p.outParents[j] = who;
      p.outTokens[j] = t;
      bool end = p.done[who] != 0;
      for (int e = 0; e < 4; ++e) end = end || (t >= 0 && t == p.eos[e]);
      p.outDone[j] = end ? 1 : 0;
    }
    if (lane == who) ++next;
  }
}

}  // namespace lkd

namespace {

int64_t beamWaves(int64_t v) { return (v + lkd::kBeamWave - 1) / lkd::kBeamWave; }

}  // namespace

extern "C" {

int64_t lk_hip_beam_select_workspace_bytes(int64_t b, int64_t v, int k) {
  if (b <= 0 || v <= 0 || k <= 0) return 0;
  const int64_t w = beamWaves(v);
  return (b * w * (8 + 8 * static_cast<int64_t>(k)) + b * k * 12 + 15) / 16 * 16;
}

int lk_hip_beam_select_f32(const float* logits, const float* scores, const int64_t* done, float* out_scores,
                           int64_t* out_parents, int64_t* out_tokens, int64_t* out_done, int64_t b, int64_t v, int k,
                           const int* eos, int num_eos, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lkd;
  if (b <= 0 || b > kBeamMost || k <= 0 || k > kBeamMost || v <= 0 || v > int64_t{kBeamWave} * kBeamLists || k > b * v ||
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
  p.waves = static_cast<int>(beamWaves(v));
  char* w = static_cast<char*>(workspace);
  p.lists = reinterpret_cast<uint2*>(w);
  w += b * p.waves * k * 8;
  p.cand = reinterpret_cast<double*>(w);
  w += b * k * 8;
  p.sums = reinterpret_cast<float*>(w);
  w += b * p.waves * 8;
  p.tok = reinterpret_cast<int*>(w);
  p.outScores = out_scores;
  p.outParents = out_parents;
  p.outTokens = out_tokens;
  p.outDone = out_done;
  p.v = v;
  p.b = static_cast<int>(b);
  p.k = k;
  for (int i = 0; i < 4; ++i) p.eos[i] = i < num_eos ? eos[i] : -1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(beamScanKernel, dim3(static_cast<unsigned>((p.waves + 3) / 4), static_cast<unsigned>(b)), dim3(256), 0, s, p);
  hipLaunchKernelGGL(beamRowKernel, dim3(static_cast<unsigned>(b)), dim3(64), static_cast<size_t>(p.waves) * k * 8, s, p);
  hipLaunchKernelGGL(beamPickKernel, dim3(1), dim3(64), 0, s, p);
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
