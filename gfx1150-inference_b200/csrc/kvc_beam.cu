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
constexpr int kPerLane = 16;                                // logits a lane holds at a time
constexpr int kBatch = 32 * kPerLane;                       // logits a warp takes at a time
constexpr int kMaxBatches = 8;                              // that a warp takes
constexpr int kMinChunk = kChunkWarps * kBatch;             // logits of one CTA, at least

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

template <typename T>
struct Pair {
  using type = float2;
};
template <>
struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ __half2 zero() { return __float2half2_rn(0.f); }
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ __nv_bfloat162 zero() { return __float2bfloat162_rn(0.f); }
};

// 16 logits of a lane, as fp32; what is not finite, and what lies past the row, is -inf.
// Which lane holds which token never depends on the row's address, so equal rows have
// equal sums.  A row that starts off a 16-byte boundary is read in aligned pairs of
// vectors and shifted into place; vectors that reach past the row go element by element.
template <typename T>
struct Batch {
  static constexpr int N = 16 / sizeof(T), V = kPerLane / N;
  union Vec {
    uint32_t w[8];
    uint4 q[2];
    T raw[2 * N];
    __device__ Vec() {}
  };
  Vec v[V];

  static __device__ __forceinline__ void load_vec(Vec& v, const T* x, int lead, int vocab, int t) {
    if (lead == 0 && t + N <= vocab) {
      v.q[0] = *reinterpret_cast<const uint4*>(x + t);
    } else if (t >= lead && t - lead + 2 * N <= vocab) {
      v.q[0] = *reinterpret_cast<const uint4*>(x + t - lead);
      v.q[1] = *reinterpret_cast<const uint4*>(x + t - lead + N);
      const int bytes = lead * static_cast<int>(sizeof(T));
      if (bytes & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) v.w[k] = v.w[k + 2];
      }
      if (bytes & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) v.w[k] = v.w[k + 1];
      }
      if (bytes & 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v.w[k] = __funnelshift_r(v.w[k], v.w[k + 1], 16);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v.raw[e] = t + e < vocab ? x[t + e] : from_f32<T>(-INFINITY);
    }
  }
  __device__ __forceinline__ void load(const T* x, int lead, int vocab, int t0) {
#pragma unroll
    for (int i = 0; i < V; ++i) load_vec(v[i], x, lead, vocab, t0 + i * 32 * N);
  }
  // the logits in fp32; returns their max
  __device__ __forceinline__ float get(float* f, bool dead) const {
    float top, odd;    // odd: NaN as soon as one is not finite
    if constexpr (sizeof(T) == 2) {
      using T2 = typename Pair<T>::type;
      T2 t2 = pair(0), z = Pair<T>::zero(), o2 = z;
#pragma unroll
      for (int k = 0; k < kPerLane / 2; ++k) {
        t2 = __hmax2(t2, pair(k));
        o2 = __hfma2(pair(k), z, o2);
      }
      top = fmaxf(to_f32<T>(t2.x), to_f32<T>(t2.y));
      odd = to_f32<T>(o2.x) + to_f32<T>(o2.y);
    } else {
      top = to_f32<T>(v[0].raw[0]);
      odd = 0.f;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const float e = to_f32<T>(v[i / N].raw[i % N]);
        top = fmaxf(top, e);
        odd = fmaf(e, 0.f, odd);
      }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) f[i] = to_f32<T>(v[i / N].raw[i % N]);
    if (dead || odd != 0.f) {
      top = -INFINITY;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        if (dead || !isfinite(f[i])) f[i] = -INFINITY;
        top = fmaxf(top, f[i]);
      }
    }
    return top;
  }
  __device__ __forceinline__ typename Pair<T>::type pair(int k) const {
    return reinterpret_cast<const typename Pair<T>::type&>(v[2 * k / N].w[2 * k % N / 2]);
  }
};

// exp(x - m), x at most m; the difference is taken first, so that nothing is lost or
// overflows where both are large.
__device__ __forceinline__ float exp_diff(float x, float m) {
  return m == -INFINITY ? 0.f : fast_exp2((x - m) * kLog2e);
}

// One CTA takes `batches` x kMinChunk logits of a row, each warp a run of its own, in one
// pass over memory that keeps a running max and sum per lane and nothing else.  The n_out-th
// largest of the 256 lanes' best then bounds the chunk's n_out best from below, and only the
// n_out lanes whose best reaches it can hold any of them: these lanes read their logits once
// more (from L2) for the few that do.  (Keeping candidates during the pass cost four times
// the instructions: nearly every batch of a run holds one that looks good so far.)
// 24 x 8 rows of 128256, fp16: 26.6 us with the join over states in turn that do not stay in
// L2, against 7.6 for the bytes; replayed on one state, which does, 17 and 5 for the join.  What
// is left are the instructions (16 per logit) and the second, partial wave of CTAs.  Runs of 4
// batches took a fifth longer than runs of 8, runs of 16 as long.
template <typename T>
__global__ void __launch_bounds__(32 * kChunkWarps) beam_chunk_kernel(const BeamArgs a) {
  // at most n_out lanes hold candidates, and each holds at most its logits
  __shared__ uint64_t s_keys[kMaxBeamOut * kPerLane * kMaxBatches];
  __shared__ uint64_t s_list[kChunkWarps][32];
  __shared__ float2 s_ml[kChunkWarps];
  __shared__ int s_holder[32 * kChunkWarps], s_holders, s_keys_n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.y;
  const int first = (blockIdx.x * kChunkWarps + warp) * a.batches * kBatch;
  const T* x = reinterpret_cast<const T*>(a.logits + static_cast<size_t>(row) * a.row_bytes);
  using B = Batch<T>;
  constexpr int N = B::N;
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  // batches of this warp that reach into the row; token of a lane's logit i of batch b
  const int batches = min(a.batches, (a.vocab - first + kBatch - 1) / kBatch);
  auto token = [&](int b, int i) { return first + b * kBatch + lane * N + (i / N) * 32 * N + i % N; };
  wait_prerequisites();
  launch_dependents();
  const bool dead = !isfinite(a.cum[row]);   // a beam that is not in use
  float m = -INFINITY, sum = 0.f;
  int at = 0;                                // the batch of the lane's best
  {
    B now, next;
    if (batches > 0) now.load(x, lead, a.vocab, token(0, 0));
    for (int b = 0; b < batches; ++b) {
      if (b + 1 < batches) next.load(x, lead, a.vocab, token(b + 1, 0));
      float f[kPerLane];
      const float top = now.get(f, dead);
      if (top > m) at = b;
      const float mm = fmaxf(m, top), ref = mm == -INFINITY ? 0.f : mm;
      float2 part = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPerLane; i += 2) {
        const float2 d = mul2(add2(make_float2(f[i], f[i + 1]), make_float2(-ref, -ref)),
                              make_float2(kLog2e, kLog2e));
        part = add2(part, make_float2(fast_exp2(d.x), fast_exp2(d.y)));
      }
      sum = sum * exp_diff(m, mm) + (part.x + part.y);
      m = mm;
      now = next;
    }
  }
  float wm = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(kAll, wm, o));
  sum *= exp_diff(m, wm);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  if (lane == 0) s_ml[warp] = make_float2(wm, sum);

  // the lane's best: the first logit of its batch that has the lane's max
  uint64_t best = 0;
  if (batches > 0) {
    B again;
    again.load(x, lead, a.vocab, token(at, 0));
    float f[kPerLane];
    again.get(f, dead);
#pragma unroll
    for (int i = kPerLane - 1; i >= 0; --i)
      if (f[i] == m && token(at, i) < a.vocab) best = make_key(m, token(at, i));
  }
  // joins the warps' descending lists; the result is warp 0's
  auto join = [&](uint64_t list) {
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
    return list;
  };
  join(sort32(best, lane));
  const uint64_t bound = s_list[0][a.n_out - 1];
  const float bound_f = bound ? from_ordered(static_cast<uint32_t>(bound >> 32)) : -INFINITY;
  if (threadIdx.x == 0) s_holders = s_keys_n = 0;
  __syncthreads();
  if (best != 0 && best >= bound) s_holder[atomicAdd(&s_holders, 1)] = threadIdx.x;
  __syncthreads();
  // the holders' vectors, spread over the CTA (their order, and the order in which hits are
  // put down, do not matter: keys are all different and get sorted)
  const int per = a.batches * B::V, holders = s_holders;
  for (int j = threadIdx.x; j < holders * per; j += 32 * kChunkWarps) {
    const int who = s_holder[j / per], q = j % per;
    const int t0 = (blockIdx.x * kChunkWarps + (who >> 5)) * a.batches * kBatch + (who & 31) * N +
                   (q / B::V) * kBatch + (q % B::V) * 32 * N;
    if (t0 >= a.vocab) continue;
    typename B::Vec v;
    B::load_vec(v, x, lead, a.vocab, t0);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float f = to_f32<T>(v.raw[e]);
      if (dead || !isfinite(f)) f = -INFINITY;
      if (t0 + e < a.vocab && f >= bound_f) {
        const uint64_t key = make_key(f, t0 + e);
        if (key >= bound) s_keys[atomicAdd(&s_keys_n, 1)] = key;
      }
    }
  }
  __syncthreads();
  uint64_t list = 0;
  const int n_keys = s_keys_n;
  for (int k = warp * 32; k < n_keys; k += 32 * kChunkWarps)
    list = merge32(list, sort32(k + lane < n_keys ? s_keys[k + lane] : 0, lane), lane);
  if (n_keys > 32) list = join(list);
  if (warp == 0) {
    const size_t slot = static_cast<size_t>(row) * a.n_chunks + blockIdx.x;
    if (lane < a.n_out) a.cand[slot * a.n_out + lane] = list;
    float2 ml = lane < kChunkWarps ? s_ml[lane] : make_float2(-INFINITY, 0.f);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    float l = ml.y * exp_diff(ml.x, top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(kAll, l, o);
    if (lane == 0) a.ml[slot] = make_float2(top, l);
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
// then the beams' lists are joined pairwise.  The join itself is in 64 bits, so it adds
// nothing to what the row sums are off by, and equal rows with equal scores tie exactly.
// The sums come in fp32 pieces.  In roundings of 2^-24: an exponential is off by 4 and by
// 2.25 per nat below the max (16 nats on the weighted average, at most, of 2^27 tokens), a
// lane's sum by 52 (4 additions of a batch, 8 batches with a factor each), its warp's and
// its chunk's by 10 each: a log sum by less than 112, which is 2^-17.  Candidates of
// different beams closer together than two of these may change places; those of one beam
// never do.
__global__ void __launch_bounds__(32 * kMaxBeams) beam_merge_kernel(const BeamArgs a) {
  wait_prerequisites();
  launch_dependents();
  __shared__ Scored s_list[kMaxBeams][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x, row = seq * a.beams + warp;
  const size_t slot0 = static_cast<size_t>(row) * a.n_chunks;
  uint64_t list = 0;
  float m = -INFINITY;
  for (int c0 = 0; c0 < a.n_chunks; c0 += 4) {   // four lists on their way at a time
    uint64_t l4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      l4[i] = c0 + i < a.n_chunks && lane < a.n_out ? a.cand[(slot0 + c0 + i) * a.n_out + lane] : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) list = merge32(list, l4[i], lane);
  }
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

int beam_chunks(int vocab) { return (vocab + kMinChunk - 1) / kMinChunk; }

// (both kernels let their successor begin only once all before them has ended)
cudaError_t launch_beam_select(BeamArgs a, cudaStream_t s) {
  // Longer runs spread a warp's sorting over more logits; shorter ones fill the GPU.
  const int rows = a.n * a.beams, most = beam_chunks(a.vocab);
  a.batches = kMaxBatches;
  while (a.batches > 1 && static_cast<int64_t>(rows) * most / a.batches < 4 * a.sms) a.batches /= 2;
  a.n_chunks = (most + a.batches - 1) / a.batches;
  const dim3 grid(static_cast<unsigned>(a.n_chunks), static_cast<unsigned>(rows));
  cudaError_t e;
  switch (a.dtype) {
    case KVC_DTYPE_F16: e = launch_early(beam_chunk_kernel<__half>, grid, 32 * kChunkWarps, 0, s, a); break;
    case KVC_DTYPE_BF16: e = launch_early(beam_chunk_kernel<__nv_bfloat16>, grid, 32 * kChunkWarps, 0, s, a); break;
    case KVC_DTYPE_F32: e = launch_early(beam_chunk_kernel<float>, grid, 32 * kChunkWarps, 0, s, a); break;
    default: return cudaErrorInvalidValue;
  }
  if (e != cudaSuccess) return e;
  return launch_early(beam_merge_kernel, dim3(static_cast<unsigned>(a.n)), 32 * a.beams, 0, s, a);
}

}  // namespace kvc
