// Kernels of a serving step around the attention itself:
//   norm_rope_kernel    RMSNorm and rotation of q and the new K heads fused with the scatter
//                       of the K/V rows into the paged pool
//   evict_select_kernel the slots that stay, by their summed attention weights
//   evict_move_kernel   their K/V rows moved together, all layers
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>

#include "kvc_device.cuh"
#include "kvc_paged.cuh"
#include "kvc_serve.h"

namespace kvc {
namespace {

// =====================================================================================
// Norm + rotate + append.  y = R(p) (x w / sqrt(mean(x^2) + eps)) for the heads of q and K,
// V as it is.  A CTA takes a token: its angles are computed once and serve all its
// heads (turns in 64 bits with the whole ones removed, then sincospif, as append_rope_kernel
// does), each pair with the position of its own axis.  A head belongs to kLanes lanes of one
// warp, each of which owns two 16-byte units that hold each other's pairs, so the sum of
// squares is a few shuffles and the head is read once.  All in 32 bits, rounded once.
//
// Bound by the chain of a CTA (its first heads and page, the angles, the stores) and by how many
// heads an SM has on their way; DRAM is at 43 % of its nominal rate.  8,634 tokens of 32 + 8 + 8
// heads of 128 dims, fp16, three axes, 43.8 us for 212 MB (32 at the copy rate; append_rope_kernel
// 45); two heads of a lane group on their way 47.4, four 47.3; fp32, with twice the bytes in the
// same chain, 70.9 (65).  An SM takes 1,024 threads (768: 47.4), which weights and angles in
// registers do not leave room for.
// =====================================================================================
constexpr int kNormThreads = 256;
constexpr int kNormBatch = 3;      // heads of a lane group on their way

template <typename T, bool kNeox, int kThreads, int kLanes>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) norm_rope_kernel(const NormRopeArgs a) {
  constexpr int kAtOnce = kThreads / kLanes, N = Unit<T>::N;
  __shared__ float4 cs[kMaxRopePairs / 2];    // two pairs' (cos, sin)
  __shared__ uint4 s_weight[2][2 * kLanes];
  __shared__ int s_page;
  const int U = a.p.row_units, Hkv = a.p.num_kv_heads, H = a.num_heads;
  const int heads = H + 2 * Hkv;                     // q, K and V heads
  const int row0 = threadIdx.x / kLanes, i = threadIdx.x % kLanes;   // first head, unit pair
  const bool works = i < U / 2;
  const int turned = a.pairs / N;                    // unit pairs that are rotated
  const bool turns = i < turned;
  // the rotated front of a NeoX head: units i and i + turned; neighbours otherwise
  const int u0 = kNeox && turns ? i : 2 * i, du = kNeox && turns ? turned : 1;
  const size_t t = blockIdx.x;
  const size_t row_bytes = static_cast<size_t>(U) * 16;
  wait_prerequisites();

  struct Item {
    Unit<T> x0, x1;
  };
  const uint8_t* q_src = a.q + t * a.q_stride + u0 * 16;
  const uint8_t* k_src = a.k_new + t * a.k_stride + u0 * 16;
  const uint8_t* v_src = a.v_new + t * a.v_stride + u0 * 16;
  auto load = [&](int head, Item& it) {
    if (!works || head >= heads) {
      it.x0.raw = it.x1.raw = make_uint4(0, 0, 0, 0);
      return;
    }
    const uint8_t* src = head < H         ? q_src + head * row_bytes
                         : head < H + Hkv ? k_src + (head - H) * row_bytes
                                          : v_src + (head - H - Hkv) * row_bytes;
    it.x0.raw = *reinterpret_cast<const uint4*>(src);
    it.x1.raw = *reinterpret_cast<const uint4*>(src + du * 16);
  };
  Item items[kNormBatch];
#pragma unroll
  for (int k = 0; k < kNormBatch; ++k) load(row0 + k * kAtOnce, items[k]);
  // (weights and angles are read where they are used: in registers they would leave an SM
  // room for fewer CTAs)
  for (int x = threadIdx.x; x < 2 * U; x += kThreads) {
    const int k = x >= U, u = x - k * U;
    const uint8_t* w = k ? a.k_weight : a.q_weight;
    if (w) s_weight[k][u] = *reinterpret_cast<const uint4*>(w + u * 16);
  }
  for (int j = threadIdx.x; j < a.pairs; j += kThreads) {
    double turn = static_cast<double>(a.rope_positions[t * a.axes + a.axis[j]]) * a.turns[j];
    turn -= rint(turn);
    // (by pairs of a unit pair, then unit pair: neighbouring threads read neighbouring angles)
    const int k = j % N;
    float2& out = reinterpret_cast<float2*>(cs + k / 2 * turned + j / N)[k & 1];
    sincospif(2.0f * static_cast<float>(turn), &out.y, &out.x);
  }
  const int pos = a.positions[t];
  if (threadIdx.x == 0) s_page = pos < 0 ? -1 : page_of(a.p, a.rows ? a.rows[t] : 0, pos);
  __syncthreads();
  const int page = s_page;
  if (page < 0) return;                              // padding, or reported
  const float4* angles = cs + i;
  uint8_t* q_dst = a.q_out + t * H * row_bytes + u0 * 16;
  const size_t place = unit_at(a.p, page, 0, pos % a.p.page_size, u0);
  const int dp = du * (a.p.layout == kLayoutCore ? 128 : 16);
  const float inv_d = 1.0f / a.head_dim;
  const int last = heads - 1;
  // (every lane of a warp goes through every round: the shuffles need them all)
  for (int h0 = row0; h0 - row0 <= last; h0 += kNormBatch * kAtOnce) {
#pragma unroll
    for (int k = 0; k < kNormBatch; ++k) {
      const int head = h0 + k * kAtOnce;
      Item& it = items[k];
      const bool is_q = head < H, is_k = !is_q && head < H + Hkv;
      const bool normed = is_q ? a.q_weight != nullptr : is_k && a.k_weight != nullptr;
      float x0[N], x1[N], scale = 1.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x0[e] = to_f32<T>(it.x0.v[e]);
        x1[e] = to_f32<T>(it.x1.v[e]);
      }
      // (a warp's heads may differ in what they need: all lanes take part in the sum)
      if (__any_sync(0xffffffffu, normed)) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          sum = fmaf(x0[e], x0[e], sum);
          sum = fmaf(x1[e], x1[e], sum);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        scale = rsqrtf(fmaf(sum, inv_d, a.eps));
      }
      if (works && head < heads) {
        if (normed) {
          Unit<T> w0, w1;
          w0.raw = s_weight[is_q ? 0 : 1][u0];
          w1.raw = s_weight[is_q ? 0 : 1][u0 + du];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            x0[e] = x0[e] * scale * to_f32<T>(w0.v[e]);
            x1[e] = x1[e] * scale * to_f32<T>(w1.v[e]);
          }
        }
        if ((is_q || is_k) && turns) {
#pragma unroll
          for (int e = 0; e < N / 2; ++e) {
            const float4 c = angles[e * turned];
            if constexpr (kNeox) {
              turn_pair(x0[2 * e], x1[2 * e], make_float2(c.x, c.y));
              turn_pair(x0[2 * e + 1], x1[2 * e + 1], make_float2(c.z, c.w));
            } else {
              // pairs 2 e and 2 e + 1 of the two units' N
              float* x = e < N / 4 ? x0 + 4 * e : x1 + 4 * e - N;
              turn_pair(x[0], x[1], make_float2(c.x, c.y));
              turn_pair(x[2], x[3], make_float2(c.z, c.w));
            }
          }
        }
        if (is_q || is_k) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            it.x0.v[e] = from_f32<T>(x0[e]);
            it.x1.v[e] = from_f32<T>(x1[e]);
          }
        }
        if (is_q) {
          uint8_t* d = q_dst + head * row_bytes;
          *reinterpret_cast<uint4*>(d) = it.x0.raw;
          *reinterpret_cast<uint4*>(d + du * 16) = it.x1.raw;
        } else {
          uint8_t* d = (is_k ? a.p.k : a.p.v) + place +
                       (head - H - (is_k ? 0 : Hkv)) * a.p.page_head_bytes;
          *reinterpret_cast<uint4*>(d) = it.x0.raw;
          *reinterpret_cast<uint4*>(d + dp) = it.x1.raw;
        }
      }
    }
    const int next = h0 + kNormBatch * kAtOnce;
#pragma unroll
    for (int k = 0; k < kNormBatch; ++k) load(next + k * kAtOnce, items[k]);
  }
}

// Any even head dim and any number of rotated pairs: a warp takes a head, a lane every 32nd
// pair of its dims.
template <typename T, bool kNeox>
__global__ void __launch_bounds__(kNormThreads) norm_rope_any_kernel(const NormRopeArgs a) {
  constexpr int N = Unit<T>::N, kHeld = kMaxRopePairs / 32;
  __shared__ float2 cs[kMaxRopePairs];
  const int Hkv = a.p.num_kv_heads, H = a.num_heads, heads = H + 2 * Hkv, half = a.head_dim / 2;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const size_t t = blockIdx.x;
  wait_prerequisites();
  for (int j = threadIdx.x; j < a.pairs; j += kNormThreads) {
    double turn = static_cast<double>(a.rope_positions[t * a.axes + a.axis[j]]) * a.turns[j];
    turn -= rint(turn);
    sincospif(2.0f * static_cast<float>(turn), &cs[j].y, &cs[j].x);
  }
  __shared__ int s_page;
  const int pos = a.positions[t];
  if (threadIdx.x == 0) s_page = pos < 0 ? -1 : page_of(a.p, a.rows ? a.rows[t] : 0, pos);
  __syncthreads();
  const int page = s_page;
  if (page < 0) return;                              // padding, or reported
  const int slot = pos % a.p.page_size;
  for (int head = warp; head < heads; head += kNormThreads / 32) {
    const bool is_q = head < H, is_k = !is_q && head < H + Hkv;
    const int h = head - (is_q ? 0 : is_k ? H : H + Hkv);
    const T* src = reinterpret_cast<const T*>(is_q   ? a.q + t * a.q_stride
                                              : is_k ? a.k_new + t * a.k_stride
                                                     : a.v_new + t * a.v_stride) +
                   static_cast<size_t>(h) * a.head_dim;
    const T* w = reinterpret_cast<const T*>(is_q ? a.q_weight : is_k ? a.k_weight : nullptr);
    auto dims = [&](int j, int& i0, int& i1) {
      const bool apart = kNeox && j < a.pairs;
      i0 = apart ? j : 2 * j;
      i1 = apart ? j + a.pairs : 2 * j + 1;
    };
    T x[kHeld][2];
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int j = lane + 32 * k;
      if (j >= half) continue;
      int i0, i1;
      dims(j, i0, i1);
      x[k][0] = src[i0];
      x[k][1] = src[i1];
      const float f0 = to_f32<T>(x[k][0]), f1 = to_f32<T>(x[k][1]);
      sum = fmaf(f0, f0, sum);
      sum = fmaf(f1, f1, sum);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float r = rsqrtf(fmaf(sum, 1.0f / a.head_dim, a.eps));
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int j = lane + 32 * k;
      if (j >= half) continue;
      int i0, i1;
      dims(j, i0, i1);
      if (is_q || is_k) {
        float f0 = to_f32<T>(x[k][0]), f1 = to_f32<T>(x[k][1]);
        if (w) {
          f0 = f0 * r * to_f32<T>(w[i0]);
          f1 = f1 * r * to_f32<T>(w[i1]);
        }
        if (j < a.pairs) turn_pair(f0, f1, cs[j]);
        x[k][0] = from_f32<T>(f0);
        x[k][1] = from_f32<T>(f1);
      }
      if (is_q) {
        T* dst = reinterpret_cast<T*>(a.q_out) + (t * H + h) * a.head_dim;
        dst[i0] = x[k][0];
        dst[i1] = x[k][1];
      } else {
        uint8_t* dst = is_k ? a.p.k : a.p.v;
        reinterpret_cast<T*>(dst + unit_at(a.p, page, h, slot, i0 / N))[i0 % N] = x[k][0];
        reinterpret_cast<T*>(dst + unit_at(a.p, page, h, slot, i1 / N))[i1 % N] = x[k][1];
      }
    }
  }
}

// Many tokens: 64 threads each (8,634 tokens, two heads on their way: 47.6 us; 32: 53, with
// two or four tokens in a CTA, which wait for one another's angles, 48.3 and 49.9); few: 256.
template <typename T, bool kNeox, int kLanes>
cudaError_t run_norm_rope(const NormRopeArgs& a, int sms, cudaStream_t s) {
  if (a.n >= 4 * sms)
    return launch_early(norm_rope_kernel<T, kNeox, 64, kLanes>, dim3(a.n), 64, 0, s, a);
  return launch_early(norm_rope_kernel<T, kNeox, kNormThreads, kLanes>, dim3(a.n), kNormThreads, 0, s, a);
}

template <typename T, bool kNeox>
cudaError_t run_norm_rope_any(const NormRopeArgs& a, int sms, cudaStream_t s) {
  const int units = a.p.row_units;
  if (units % 2 == 0 && a.pairs % Unit<T>::N == 0) {
    if (units <= 8) return run_norm_rope<T, kNeox, 4>(a, sms, s);
    if (units <= 16) return run_norm_rope<T, kNeox, 8>(a, sms, s);
    if (units <= 32) return run_norm_rope<T, kNeox, 16>(a, sms, s);
    return run_norm_rope<T, kNeox, 32>(a, sms, s);
  }
  return launch_early(norm_rope_any_kernel<T, kNeox>, dim3(a.n), kNormThreads, 0, s, a);
}

template <typename T>
cudaError_t run_norm_rope_type(const NormRopeArgs& a, bool neox, int sms, cudaStream_t s) {
  return neox ? run_norm_rope_any<T, true>(a, sms, s) : run_norm_rope_any<T, false>(a, sms, s);
}

// =====================================================================================
// Which slots stay.  A CTA takes one (layer, sequence, KV head): of the slots in front of
// the last `recent` it keeps the budget - recent heaviest, equal ones from the lowest slot on.
//
// The weight on the border is found in three steps over weights that wait in shared memory: a
// histogram of their upper 11 bits (sign, exponent, two more) names the bin it is in, that
// bin's weights are put on a list, and every thread counts how many of the list are above the
// one that it takes.  (A list of more than kSelectList, as equal weights make it, is searched
// seven bits at a time instead.)  One ordered pass then writes the kept slots and their weights,
// which may go to where they came from: a slot never moves up, and all weights of a round are
// read before any of it is written.  Bound by latency where there are few heads (88 of 600
// weights: 6.7 us; 8.8 with four passes of eight bits), by its instructions and barriers where
// there are many (2,048 of 900-3,100: 38 us, issue slots 60 % busy; 36 with the passes).
// =====================================================================================
constexpr int kSelectThreads = 256;
constexpr int kSelectHeld = 8192;    // weights kept in shared memory; longer rows are read again
constexpr int kSelectBins = 2048;
constexpr int kSelectList = 256;
constexpr int kSelectPer = 4;        // slots of a thread in a round of the ordered pass

// Larger for a larger weight; what is not a number comes last.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);   // (-0 ties with 0)
  return w != w ? 0u : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
  extern __shared__ float s_w[];
  __shared__ uint32_t s_hist[kSelectBins];
  __shared__ uint32_t s_list[kSelectList];
  __shared__ uint32_t s_digit, s_need, s_listed, s_ties;
  constexpr int kWarps = kSelectThreads / 32, kBinsPer = kSelectBins / kSelectThreads;
  __shared__ int s_warp[2][kWarps];
  const int head = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z;
  const int Hkv = a.p.num_kv_heads, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_prerequisites();
  const int n = a.ctx[seq], row = a.rows ? a.rows[seq] : seq;
  int32_t* kept = a.kept + ((static_cast<size_t>(layer) * a.n + seq) * Hkv + head) * a.budget;
  const bool fits = row >= 0 && row < a.p.bt_rows && row < a.weight_rows && n >= 0 &&
                    n <= a.weight_slots && n <= static_cast<int64_t>(a.p.bt_stride) * a.p.page_size;
  if (!fits) {
    if (tid == 0) report_error_at(a.p.err, KVC_DEVERR_BAD_POSITION, static_cast<uint32_t>(n));
    for (int j = tid; j < a.budget; j += kSelectThreads) kept[j] = -1;
    return;
  }
  const size_t base = ((static_cast<size_t>(layer) * a.weight_rows + row) * Hkv + head) * a.weight_slots;
  const float* w = a.weights + base;
  float* left = a.weights_out + base;
  if (n <= a.budget) {
    for (int j = tid; j < a.budget; j += kSelectThreads) {
      kept[j] = j < n ? j : -1;
      if (j < n && left != w) left[j] = w[j];
    }
    return;
  }
  const int old = n - a.recent, take = a.budget - a.recent;   // take of [0, old), all behind
  const bool held = old <= kSelectHeld;
  auto weight = [&](int i) { return held ? s_w[i] : w[i]; };
  // How many of the largest are still wanted of the bins [0, bins) of s_hist, and in which of
  // them the last one is: s_need, s_digit.  All threads; the bins are zero afterwards.
  auto find = [&](uint32_t need, int bins) {
    uint32_t cnt[kBinsPer], mine = 0;
#pragma unroll
    for (int b = 0; b < kBinsPer; ++b) {
      const int bin = tid * kBinsPer + b;
      cnt[b] = bin < bins ? s_hist[bin] : 0u;
      if (bin < bins) s_hist[bin] = 0;
      mine += cnt[b];
    }
    uint32_t above = mine;                                    // of this lane's bins and those above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_down_sync(0xffffffffu, above, o);
      if (lane + o < 32) above += v;
    }
    if (lane == 0) s_warp[0][warp] = static_cast<int>(above);
    __syncthreads();
    uint32_t over = above - mine;
    for (int x = warp + 1; x < kWarps; ++x) over += s_warp[0][x];
    if (over < need && need <= over + mine) {
      bool found = false;
#pragma unroll
      for (int b = kBinsPer - 1; b >= 0; --b) {
        if (!found && need <= over + cnt[b]) {
          s_digit = tid * kBinsPer + b;
          s_need = need - over;
          s_ties = cnt[b];
          found = true;
        }
        over += cnt[b];
      }
    }
    __syncthreads();
  };
  uint32_t border = 0, need = 0, ties_all = 0;                // kept: above border, and `need` on it
  if (take > 0) {
    for (int b = tid; b < kSelectBins; b += kSelectThreads) s_hist[b] = 0;
    if (tid == 0) s_listed = 0;
    __syncthreads();
    for (int i0 = tid; i0 < old; i0 += 8 * kSelectThreads) {  // eight on their way
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = i0 + k * kSelectThreads < old ? w[i0 + k * kSelectThreads] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + k * kSelectThreads;
        if (i >= old) break;
        if (held) s_w[i] = v[k];
        atomicAdd(&s_hist[weight_key(v[k]) >> 21], 1u);
      }
    }
    __syncthreads();
    find(take, kSelectBins);
    const uint32_t top = s_digit;
    need = s_need;
    ties_all = s_ties;
    if (ties_all <= kSelectList) {
      for (int i = tid; i < old; i += kSelectThreads) {
        const uint32_t k = weight_key(weight(i));
        if (k >> 21 == top) s_list[atomicAdd(&s_listed, 1u)] = k;
      }
      __syncthreads();
      if (tid < ties_all) {
        const uint32_t k = s_list[tid];
        uint32_t over = 0, same = 0;
        for (uint32_t x = 0; x < ties_all; ++x) {
          const uint32_t y = s_list[x];
          over += y > k;
          same += y == k;
        }
        if (over < need && need <= over + same) {             // (all equal ones write the same)
          s_digit = k;
          s_need = need - over;
          s_ties = same;
        }
      }
      __syncthreads();
      border = s_digit;
    } else {
      border = top << 21;
      for (int shift = 14; shift >= 0; shift -= 7) {
        for (int i = tid; i < old; i += kSelectThreads) {
          const uint32_t k = weight_key(weight(i));
          if (k >> (shift + 7) == border >> (shift + 7)) atomicAdd(&s_hist[(k >> shift) & 127u], 1u);
        }
        __syncthreads();
        find(need, 128);
        border |= s_digit << shift;
        need = s_need;
      }
    }
    need = s_need;
    ties_all = s_ties;
  }
  // In order.  Where every weight on the border is kept, one comparison tells; `at` slots are
  // kept so far, and `ties` on the border were seen.
  const int limit = static_cast<int>(need);
  const bool plain = need == ties_all;
  int at = 0, ties = 0;
  for (int i0 = 0; i0 < old && take > 0; i0 += kSelectPer * kSelectThreads) {
    const int first = i0 + warp * kSelectPer * 32 + lane;     // a warp's slots are neighbours
    float v[kSelectPer];
    uint32_t over[kSelectPer], tie[kSelectPer];
    int n_over = 0, n_tie = 0;
#pragma unroll
    for (int e = 0; e < kSelectPer; ++e) {
      const int i = first + 32 * e;
      v[e] = i < old ? weight(i) : 0.f;
      const uint32_t k = weight_key(v[e]);
      over[e] = __ballot_sync(0xffffffffu, i < old && (plain ? k >= border : k > border));
      tie[e] = plain ? 0u : __ballot_sync(0xffffffffu, i < old && k == border);
      n_over += __popc(over[e]);
      n_tie += __popc(tie[e]);
    }
    if (lane == 0) {
      s_warp[0][warp] = n_over;
      s_warp[1][warp] = n_tie;
    }
    __syncthreads();                                          // (and the round's weights are read)
    int my_over = at, my_tie = ties, all_over = 0, all_tie = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const int o = s_warp[0][x], t = s_warp[1][x];
      if (x < warp) {
        my_over += o;
        my_tie += t;
      }
      all_over += o;
      all_tie += t;
    }
    const int taken = min(ties, limit);                       // ties that were kept so far
    const uint32_t below = (1u << lane) - 1u;
#pragma unroll
    for (int e = 0; e < kSelectPer; ++e) {
      const int o = my_over + __popc(over[e] & below), t = my_tie + __popc(tie[e] & below);
      if ((over[e] >> lane & 1u) || ((tie[e] >> lane & 1u) && t < limit)) {
        const int j = o + (plain ? 0 : min(t, limit) - taken);
        kept[j] = first + 32 * e;
        left[j] = v[e];
      }
      my_over += __popc(over[e]);
      my_tie += __popc(tie[e]);
    }
    at += all_over + (plain ? 0 : min(ties + all_tie, limit) - taken);
    ties += all_tie;
    __syncthreads();
  }
  for (int i0 = 0; i0 < a.recent; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const float wi = i < a.recent ? w[old + i] : 0.f;
    __syncthreads();
    if (i < a.recent) {
      kept[take + i] = old + i;
      left[take + i] = wi;
    }
  }
}

// =====================================================================================
// The kept rows move together.  A CTA takes some of the 16-byte columns of one head of one
// layer's K or V and goes through the kept slots in order, a chunk at a time.  A slot never
// moves up, so a later chunk's sources lie behind every place written before it: the next
// chunk is read before this one is written, and only the reads of one chunk have to be done
// (a barrier) before its first write.  Rows that stay where they are are not touched.
//
// Bound by memory traffic, which is more than the rows' bytes: a row's 16-byte pieces stand
// 128 bytes apart, eight positions to a line, so of 64 bytes that memory reads at a time half
// are another row's where every second slot stays.  8 sequences of 900-3,100 cut to 1024 in 32
// layers of 8 x 128 dims, bf16: 404 us for 1.9 GB of rows, which are 2.7 GB of traffic at 6.7
// TB/s, the rate of a copy.  (Offsets of a thread's units kept in registers, places as 32-bit
// units: 475 us with divisions by the unit count in every chunk.)
// =====================================================================================
constexpr int kMoveThreads = 256;
constexpr int kMoveUnits = 8;        // 16-byte units of a thread on their way
constexpr int kMoveRows = 256;       // rows of a chunk at most

__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a, const int parts) {
  __shared__ uint2 s_place[3][kMoveRows];  // 16-byte units: where a row is and goes
  constexpr uint32_t kNone = ~0u;
  const int seq = blockIdx.y, tid = threadIdx.x;
  const int part = blockIdx.x % parts, head = blockIdx.x / parts, kv = blockIdx.z & 1, layer = blockIdx.z >> 1;
  const int Hkv = a.p.num_kv_heads, U = a.p.row_units / parts, ps = a.p.page_size;
  wait_prerequisites();
  const int n = a.ctx[seq], m = a.budget, row = a.rows ? a.rows[seq] : seq;
  const int32_t* kept = a.kept + ((static_cast<size_t>(layer) * a.n + seq) * Hkv + head) * m;
  if (n <= m) return;                      // nothing leaves
  const bool core = a.p.layout == kLayoutCore;
  uint8_t* base = (kv ? a.p.v : a.p.k) + static_cast<size_t>(layer) * a.layer_bytes;
  int chunk = kMoveThreads * kMoveUnits / U;                 // rows of a chunk
  chunk = chunk > kMoveRows ? kMoveRows : (chunk & ~7);
  const int chunks = (m + chunk - 1) / chunk;
  auto place = [&](int pos) {
    const int page = page_of(a.p, row, pos);
    return page < 0 ? kNone : static_cast<uint32_t>(unit_at(a.p, page, head, pos % ps, part * U) / 16);
  };
  auto places = [&](int c) {               // where chunk c's rows are and go
    for (int r = tid; r < chunk && c < chunks; r += kMoveThreads) {
      const int j = c * chunk + r, from = j < m ? kept[j] : j;   // (-1: reported)
      uint2 x = make_uint2(kNone, kNone);
      if (from > j) x = make_uint2(place(from), place(j));
      if (x.y == kNone) x.x = kNone;
      s_place[c % 3][r] = x;
    }
  };
  // A thread's units of a chunk, in the order of memory: row, and offset from the row's place.
  int unit[kMoveUnits];
#pragma unroll
  for (int k = 0; k < kMoveUnits; ++k) {
    const int x = tid + k * kMoveThreads, y = core ? x >> 3 : x;
    const int q = y / U, u = y - q * U, r = core ? q * 8 + (x & 7) : q;
    unit[k] = x < chunk * U ? (r << 16) | (core ? 8 * u : u) : -1;
  }
  uint4 now[kMoveUnits], next[kMoveUnits];
  auto load = [&](int c, uint4* v) {
    if (c >= chunks) return;
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) {
      if (unit[k] < 0) continue;
      const uint32_t at = s_place[c % 3][unit[k] >> 16].x;
      if (at != kNone) v[k] = reinterpret_cast<const uint4*>(base)[static_cast<size_t>(at) + (unit[k] & 0xffff)];
    }
  };
  places(0);
  places(1);
  __syncthreads();
  load(0, now);
  for (int c = 0; c < chunks; ++c) {
    __syncthreads();                       // chunk c has been read, chunk c - 1 written
    places(c + 2);
    load(c + 1, next);
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) {
      if (unit[k] < 0) continue;
      const uint2 at = s_place[c % 3][unit[k] >> 16];
      if (at.x != kNone) reinterpret_cast<uint4*>(base)[static_cast<size_t>(at.y) + (unit[k] & 0xffff)] = now[k];
    }
#pragma unroll
    for (int k = 0; k < kMoveUnits; ++k) now[k] = next[k];
  }
}

}  // namespace

// (No kernel here lets its successor begin early: they write K/V rows, and a decode two
// launches on may stream those as soon as the launch between them has begun.)

cudaError_t launch_norm_rope(const NormRopeArgs& a, int dtype, bool neox, int sms, cudaStream_t s) {
  switch (dtype) {
    case KVC_DTYPE_F16: return run_norm_rope_type<__half>(a, neox, sms, s);
    case KVC_DTYPE_BF16: return run_norm_rope_type<__nv_bfloat16>(a, neox, sms, s);
    case KVC_DTYPE_F32: return run_norm_rope_type<float>(a, neox, sms, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_evict(const EvictArgs& a, int sms, cudaStream_t s) {
  const size_t held = sizeof(float) * std::min(kSelectHeld, a.weight_slots);
  cudaError_t e = launch_early(evict_select_kernel,
                               dim3(static_cast<unsigned>(a.p.num_kv_heads), static_cast<unsigned>(a.n),
                                    static_cast<unsigned>(a.n_layers)),
                               kSelectThreads, held, s, a);
  if (e != cudaSuccess) return e;
  // few heads: their columns are spread over more CTAs
  const int64_t heads = 2ll * a.n_layers * a.n * a.p.num_kv_heads;
  int parts = 1;
  while (heads * parts < 2 * sms && a.p.row_units % (2 * parts) == 0) parts *= 2;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.p.num_kv_heads * parts), static_cast<unsigned>(a.n),
                     static_cast<unsigned>(2 * a.n_layers));
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, a, parts);
}

}  // namespace kvc
