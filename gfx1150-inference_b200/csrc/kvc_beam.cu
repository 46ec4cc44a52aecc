// Beam search's selection: the n_out best of beams x vocabulary by accumulated
// score + log softmax of the logits.
//
//   beam_chunk_kernel   one pass over the logits: per chunk of a row the max, the sum
//                       of exp(x - max) and the n_out best tokens
//   beam_merge_kernel   per sequence: the rows' log sums, and the best of all chunks
//
// Within a row the order of scores is the order of its logits, so the first pass
// needs no log sum: a candidate is a 64-bit key, (ordered bits of the logit, ~token),
// whose order is "larger logit, then lower token".  Lists of candidates are held
// sorted, one entry per lane: 32 lanes keep n_out <= 32 of them.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kvc_device.cuh"
#include "kvc_spec.h"
#include "kvcache.h"

namespace kvc {
namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kChunkWarps = 8;
constexpr int kPerLane = 16;                                // logits a lane holds
constexpr int kWarpSpan = 32 * kPerLane;
constexpr int kChunk = kChunkWarps * kWarpSpan;             // logits of one CTA

// Bits of a finite float or -inf that order like the value.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ uint64_t make_key(float x, int token) {
  x += 0.0f;  // -0 and 0 are equal logits
  return (static_cast<uint64_t>(ordered(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(token));
}

__device__ __forceinline__ uint64_t keep(uint64_t mine, uint64_t other, bool larger) {
  return (mine > other) == larger ? mine : other;
}
// 32 keys, one per lane, into descending order.
__device__ __forceinline__ uint64_t sort32(uint64_t key, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1)
      key = keep(key, __shfl_xor_sync(kAll, key, j), ((lane & j) == 0) == ((lane & k) == 0));
  return key;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
  const uint64_t r = __shfl_sync(kAll, b, 31 - lane);
  uint64_t key = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1)
    key = keep(key, __shfl_xor_sync(kAll, key, j), (lane & j) == 0);
  return key;
}

// A chunk: every lane holds kPerLane logits.  The n_out-th largest of the 32 lanes'
// best is a bound that at least n_out logits of the warp reach, and only lanes whose
// best reaches it hold any: few logits are sorted.
template <typename T>
__global__ void __launch_bounds__(32 * kChunkWarps) beam_chunk_kernel(const BeamArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ uint64_t s_pend[kChunkWarps][64];
  __shared__ uint64_t s_list[kChunkWarps][32];
  __shared__ float2 s_ml[kChunkWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y;
  const int first = blockIdx.x * kChunk + warp * kWarpSpan;
  const T* x = reinterpret_cast<const T*>(a.logits + static_cast<size_t>(row) * a.row_bytes);
  constexpr int N = 16 / sizeof(T);
  // Which lane holds which token never depends on the row's address, so equal rows have
  // equal sums.  A row that starts off a 16-byte boundary is read in aligned pairs of
  // vectors and shifted into place; vectors that reach past the row go element by element.
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  float v[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane / N; ++i) {
    const int t0 = first + (i * 32 + lane) * N;
    union {
      uint32_t w[8];
      uint4 q[2];
      T raw[2 * N];
    };
    if (lead == 0 && t0 + N <= a.vocab) {
      q[0] = __ldcs(reinterpret_cast<const uint4*>(x + t0));
    } else if (t0 >= lead && t0 - lead + 2 * N <= a.vocab) {
      q[0] = *reinterpret_cast<const uint4*>(x + t0 - lead);
      q[1] = *reinterpret_cast<const uint4*>(x + t0 - lead + N);
      const int bytes = lead * static_cast<int>(sizeof(T));
      if (bytes & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
      }
      if (bytes & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
      }
      if (bytes & 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) raw[e] = t0 + e < a.vocab ? x[t0 + e] : from_f32<T>(0.f);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) v[i * N + e] = to_f32<T>(raw[e]);
  }
  // a beam that is not in use: its candidates all score -inf
  const bool dead = !isfinite(a.cum[row]);
  uint64_t best = 0;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int t = first + ((i / N) * 32 + lane) * N + i % N;
    if (dead || !isfinite(v[i])) v[i] = -INFINITY;
    if (t < a.vocab) {
      mx = fmaxf(mx, v[i]);
      const uint64_t key = make_key(v[i], t);
      best = key > best ? key : best;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, o));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int t = first + ((i / N) * 32 + lane) * N + i % N;
    if (t < a.vocab && v[i] != -INFINITY) sum += fast_exp2((v[i] - mx) * kLog2e);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  if (lane == 0) s_ml[warp] = make_float2(mx, sum);

  const uint64_t bound = __shfl_sync(kAll, sort32(best, lane), a.n_out - 1);
  uint64_t list = 0;
  int pending = 0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int t = first + ((i / N) * 32 + lane) * N + i % N;
    const uint64_t key = t < a.vocab ? make_key(v[i], t) : 0;
    const bool in = key != 0 && key >= bound;
    const unsigned hits = __ballot_sync(kAll, in);
    if (hits == 0) continue;
    if (in) s_pend[warp][pending + __popc(hits & ((1u << lane) - 1u))] = key;
    pending += __popc(hits);
    __syncwarp();
    if (pending >= 32) {
      list = merge32(list, sort32(s_pend[warp][lane], lane), lane);
      pending -= 32;
      const uint64_t rest = s_pend[warp][32 + lane];
      __syncwarp();
      s_pend[warp][lane] = rest;
      __syncwarp();
    }
  }
  if (pending > 0) list = merge32(list, sort32(lane < pending ? s_pend[warp][lane] : 0, lane), lane);
  s_list[warp][lane] = list;
  __syncthreads();
#pragma unroll
  for (int half = kChunkWarps / 2; half > 0; half >>= 1) {
    if (warp < half) {
      list = merge32(list, s_list[warp + half][lane], lane);
      s_list[warp][lane] = list;
    }
    __syncthreads();
  }
  if (warp == 0) {
    const size_t slot = static_cast<size_t>(row) * a.n_chunks + blockIdx.x;
    if (lane < a.n_out) a.cand[slot * a.n_out + lane] = list;
    float2 ml = lane < kChunkWarps ? s_ml[lane] : make_float2(-INFINITY, 0.f);
    float m = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    float l = ml.y > 0.f ? ml.y * fast_exp2((ml.x - m) * kLog2e) : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(kAll, l, o);
    if (lane == 0) a.ml[slot] = make_float2(m, l);
  }
}

// A scored candidate; larger: better score, then lower (beam, token).
struct Scored {
  double score;
  uint32_t id;   // beam << 27 | token
};
__device__ __forceinline__ bool better(const Scored& x, const Scored& y) {
  return x.score > y.score || (x.score == y.score && x.id < y.id);
}
__device__ __forceinline__ Scored shfl_xor(const Scored& s, int j) {
  return {__shfl_xor_sync(kAll, s.score, j), __shfl_xor_sync(kAll, s.id, j)};
}
__device__ __forceinline__ Scored merge32(Scored x, const Scored& y, int lane) {
  const Scored r = {__shfl_sync(kAll, y.score, 31 - lane), __shfl_sync(kAll, y.id, 31 - lane)};
  if (better(r, x)) x = r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const Scored o = shfl_xor(x, j);
    if (better(o, x) == ((lane & j) == 0)) x = o;
  }
  return x;
}

// One CTA per sequence, one warp per beam: the warp joins its row's lists and sums,
// then the beams' lists are joined pairwise.  Scores are held in 64 bits so that
// candidates of different beams that lie close together keep their order.
__global__ void __launch_bounds__(32 * kMaxBeams) beam_merge_kernel(const BeamArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ Scored s_list[kMaxBeams][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x, row = seq * a.beams + warp;
  const size_t slot0 = static_cast<size_t>(row) * a.n_chunks;
  uint64_t list = 0;
  float m = -INFINITY;
  for (int c = 0; c < a.n_chunks; ++c)
    list = merge32(list, lane < a.n_out ? a.cand[(slot0 + c) * a.n_out + lane] : 0, lane);
  for (int c = lane; c < a.n_chunks; c += 32) m = fmaxf(m, a.ml[slot0 + c].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
  double sum = 0.0;
  for (int c = lane; c < a.n_chunks; c += 32) {
    const float2 ml = a.ml[slot0 + c];
    if (ml.y > 0.f) sum += static_cast<double>(ml.y) * exp(static_cast<double>(ml.x) - m);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  const float x = from_ordered(static_cast<uint32_t>(list >> 32));
  Scored s;
  s.score = -INFINITY;
  s.id = 0xffffffffu;
  if (list != 0) {
    s.id = (static_cast<uint32_t>(warp) << 27) | (0xffffffffu - static_cast<uint32_t>(list));
    const float cum = a.cum[row];
    if (isfinite(x) && isfinite(cum)) s.score = static_cast<double>(cum) + (static_cast<double>(x) - m - log(sum));
  }
  s_list[warp][lane] = s;
  __syncthreads();
  int n = a.beams;
  while (n > 1) {
    const int half = (n + 1) / 2;
    if (warp + half < n) {
      s = merge32(s, s_list[warp + half][lane], lane);
      s_list[warp][lane] = s;
    }
    __syncthreads();
    n = half;
  }
  if (warp == 0 && lane < a.n_out) {
    const size_t at = static_cast<size_t>(seq) * a.n_out + lane;
    a.tokens[at] = static_cast<int32_t>(s.id & ((1u << 27) - 1u));
    a.parents[at] = static_cast<int32_t>(s.id >> 27);
    a.scores[at] = static_cast<float>(s.score);
  }
}

}  // namespace

int beam_chunks(int vocab, int) { return (vocab + kChunk - 1) / kChunk; }

cudaError_t launch_beam_select(const BeamArgs& a, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>(a.n_chunks), static_cast<unsigned>(a.n * a.beams));
  switch (a.dtype) {
    case KVC_DTYPE_F16: beam_chunk_kernel<__half><<<grid, 32 * kChunkWarps, 0, s>>>(a); break;
    case KVC_DTYPE_BF16: beam_chunk_kernel<__nv_bfloat16><<<grid, 32 * kChunkWarps, 0, s>>>(a); break;
    case KVC_DTYPE_F32: beam_chunk_kernel<float><<<grid, 32 * kChunkWarps, 0, s>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.n));
  cfg.blockDim = dim3(static_cast<unsigned>(32 * a.beams));
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, beam_merge_kernel, a);
}

}  // namespace kvc
