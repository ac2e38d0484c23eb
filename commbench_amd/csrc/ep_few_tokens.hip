// The whole expert layer for a few tokens in two kernels, for gfx950:
//   act[r, i] = silu(Wg[e] x[t])[i] * (Wu[e] x[t])[i]                     r = route (t, k) to expert e
//   out[t, :] = sum_k w[t, k] * W2[e_k] act[(t, k), :] (+ biases)
// With a few tokens every expert sees one or a handful of rows, so the time is that of reading the met
// experts' weights once; moving rows to the experts and back would only add launches.  Weights are
// bf16, or int8 with a scale for each output channel (widened to bf16 in registers, exactly), products
// run on the matrix units with the weights as the 16-row operand and up to 16 of an expert's routes as
// the columns, sums are fp32.  act is rounded to bf16, the type the many-token path hands on there too.
// A sum never depends on the order in which waves finish: each (route, output) has one writer, and the
// slots of a token are added in ascending order at the end.
#include "ep_device.h"

namespace mi_ep {
namespace {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kFirstThreads = 256, kFirstWaves = kFirstThreads / kWave;
constexpr int kSecondThreads = 512, kSecondWaves = kSecondThreads / kWave;

// 8 of the int8 codes in two words as bf16 (every code is one exactly).
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  uint32_t f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t word = j < 4 ? lo : hi;
    f[j] = __float_as_uint(static_cast<float>(static_cast<int>(word << (24 - 8 * (j & 3))) >> 24));
  }
  union {
    uint32_t u[4];
    bf16x8 b;
  } out;
#pragma unroll
  for (int j = 0; j < 4; ++j) out.u[j] = __builtin_amdgcn_perm(f[2 * j + 1], f[2 * j], 0x07060302u);
  return out.b;
}
__device__ __forceinline__ bf16x8 as_bf16(vec16 v) {
  union {
    vec16 u;
    bf16x8 b;
  } out;
  out.u = v;
  return out.b;
}

// acc += W[16 rows][k] * X[16 columns][k] over the 16-byte pieces of a lane.  `w` points at the lane's
// row (lane % 16) of the weights, `x` at its column's vector; a lane without a column has x == nullptr.
// The lanes' order over k is the same on both sides, which is all a product needs.
template <bool kInt8>
struct Piece {  // elements of k that 64 lanes take in one step: 4 lane groups of 16 bytes of weights
  static constexpr int kLane = kInt8 ? 16 : 8;
  static constexpr int kStep = 4 * kLane;
};

template <bool kInt8>
__device__ __forceinline__ float4v multiply(vec16 w, const vec16* x, float4v acc) {
  const vec16 zero = {0, 0, 0, 0};
  const vec16 x0 = x != nullptr ? x[0] : zero;
  if constexpr (kInt8) {
    const vec16 x1 = x != nullptr ? x[1] : zero;
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[0], w[1]), as_bf16(x0), acc, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[2], w[3]), as_bf16(x1), acc, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(w), as_bf16(x0), acc, 0, 0, 0);
  }
}

// The routes of expert e among ids[0, count), in order, into list; returns how many (wave-uniform).
__device__ __forceinline__ int collect_routes(const int* ids, int count, int e, uint16_t* list) {
  const int lane = lane_id();
  int n = 0;
  for (int base = 0; base < count; base += kWave) {
    const bool match = base + lane < count && ids[base + lane] == e;
    const uint64_t mask = __ballot(match);
    if (match) list[n + __popcll(mask & lanes_below(lane))] = static_cast<uint16_t>(base + lane);
    n += __popcll(mask);
  }
  return n;
}

__device__ __forceinline__ void load_ids(const FewTokensArgs& a, int routes, int* ids) {
  for (int r = static_cast<int>(threadIdx.x); r < routes; r += static_cast<int>(blockDim.x)) {
    const int64_t e = a.topk_idx[r];
    ids[r] = e >= 0 && e < a.num_experts ? static_cast<int>(e) : -1;
  }
}

// Workgroup (s, r): 16 columns of act for the expert of route r, if r is that expert's first route.
template <bool kInt8>
__global__ __launch_bounds__(kFirstThreads) void ep_few_tokens_gate_up_kernel(const FewTokensArgs a) {
  __shared__ int ids[kFewRoutes];
  __shared__ uint16_t list[kFewRoutes];
  __shared__ int count;
  __shared__ float partial[kFirstWaves][2][4][kWave];
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  const int routes = a.num_tokens * a.num_topk;
  const int r = static_cast<int>(blockIdx.y);
  load_ids(a, routes, ids);
  __syncthreads();
  const int e = ids[r];
  int earlier = e < 0 ? 1 : 0;
  for (int q = static_cast<int>(threadIdx.x); q < r; q += kFirstThreads) earlier |= ids[q] == e ? 1 : 0;
  if (__syncthreads_or(earlier)) return;
  if (wave == 0) {
    const int n = collect_routes(ids, routes, e, list);
    if (lane == 0) count = n;
  }
  __syncthreads();

  const int H = a.hidden, I = a.intermediate;
  const int i0 = static_cast<int>(blockIdx.x) * 16;
  constexpr int kBytes = kInt8 ? 1 : 2;
  const int k_lane = (lane >> 4) * Piece<kInt8>::kLane;
  const unsigned char* gate = a.w13 + ((static_cast<size_t>(e) * 2 * I + i0 + (lane & 15)) * H + k_lane) * kBytes;
  const unsigned char* up = gate + static_cast<size_t>(I) * H * kBytes;
  for (int c0 = 0; c0 < count; c0 += 16) {
    const int column = c0 + (lane & 15);
    const uint16_t* x = column < count ? a.x + static_cast<size_t>(list[column] / a.num_topk) * H + k_lane : nullptr;
    float4v g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
    for (int k = wave * Piece<kInt8>::kStep; k < H; k += kFirstWaves * Piece<kInt8>::kStep) {
      const bool inside = k + k_lane < H;
      const vec16 zero = {0, 0, 0, 0};
      const vec16 wg = inside ? *reinterpret_cast<const vec16*>(gate + static_cast<size_t>(k) * kBytes) : zero;
      const vec16 wu = inside ? *reinterpret_cast<const vec16*>(up + static_cast<size_t>(k) * kBytes) : zero;
      const vec16* xk = inside && x != nullptr ? reinterpret_cast<const vec16*>(x + k) : nullptr;
      g = multiply<kInt8>(wg, xk, g);
      u = multiply<kInt8>(wu, xk, u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      partial[wave][0][i][lane] = g[i];
      partial[wave][1][i][lane] = u[i];
    }
    __syncthreads();
    if (wave == 0 && column < count) {
      float o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float gs = 0.0f, us = 0.0f;
#pragma unroll
        for (int w = 0; w < kFirstWaves; ++w) {
          gs += partial[w][0][i][lane];
          us += partial[w][1][i][lane];
        }
        if constexpr (kInt8) {
          const float* scales = a.w13_scales + static_cast<size_t>(e) * 2 * I + i0 + (lane >> 4) * 4 + i;
          gs *= scales[0];
          us *= scales[I];
        }
        o[i] = gs / (1.0f + __expf(-gs)) * us;
      }
      *reinterpret_cast<uint2*>(a.act + static_cast<size_t>(list[column]) * I + i0 + (lane >> 4) * 4) =
          uint2{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
    }
    __syncthreads();
  }
}

// Workgroup h: 16 columns of the output for every token.  The waves share out the met experts (and, with
// fewer experts than waves, ranges of the intermediate axis); y[split][route][16] collects their products.
template <bool kInt8>
__global__ __launch_bounds__(kSecondThreads) void ep_few_tokens_down_kernel(const FewTokensArgs a, const int splits) {
  extern __shared__ float y[];
  const int routes = a.num_tokens * a.num_topk;
  int* ids = reinterpret_cast<int*>(y + static_cast<size_t>(splits) * routes * 16);
  uint16_t* leaders = reinterpret_cast<uint16_t*>(ids + routes);
  uint16_t* lists = leaders + routes;  // [kSecondWaves][routes]
  __shared__ int met;
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  load_ids(a, routes, ids);
  __syncthreads();
  if (wave == 0) {  // the first route of every met expert, in order
    int n = 0;
    for (int base = 0; base < routes; base += kWave) {
      const int r = base + lane;
      bool first = r < routes && ids[r] >= 0;
      if (first)
        for (int q = 0; q < r; ++q) first = first && ids[q] != ids[r];
      const uint64_t mask = __ballot(first);
      if (first) leaders[n + __popcll(mask & lanes_below(lane))] = static_cast<uint16_t>(r);
      n += __popcll(mask);
    }
    if (lane == 0) met = n;
  }
  __syncthreads();

  const int H = a.hidden, I = a.intermediate;
  const int h0 = static_cast<int>(blockIdx.x) * 16;
  constexpr int kBytes = kInt8 ? 1 : 2;
  constexpr int kStep = Piece<kInt8>::kStep;
  const int k_lane = (lane >> 4) * Piece<kInt8>::kLane;
  const int steps = (I + kStep - 1) / kStep;
  uint16_t* list = lists + wave * routes;
  for (int item = wave; item < met * splits; item += kSecondWaves) {
    const int leader = item / splits, split = item - leader * splits;
    const int e = ids[leaders[leader]];
    const int count = collect_routes(ids, routes, e, list);
    const int k_begin = steps * split / splits * kStep, k_end = steps * (split + 1) / splits * kStep;
    const unsigned char* w = a.w2 + ((static_cast<size_t>(e) * H + h0 + (lane & 15)) * I + k_lane) * kBytes;
    for (int c0 = 0; c0 < count; c0 += 16) {
      const int column = c0 + (lane & 15);
      const int route = column < count ? list[column] : 0;
      const uint16_t* x = column < count ? a.act + static_cast<size_t>(route) * I + k_lane : nullptr;
      float4v acc = {0, 0, 0, 0};
      for (int k = k_begin; k < k_end; k += kStep) {
        const bool inside = k + k_lane < I;
        const vec16 zero = {0, 0, 0, 0};
        const vec16 wk = inside ? *reinterpret_cast<const vec16*>(w + static_cast<size_t>(k) * kBytes) : zero;
        acc = multiply<kInt8>(wk, inside && x != nullptr ? reinterpret_cast<const vec16*>(x + k) : nullptr, acc);
      }
      if (column < count) {
        float* out = y + (static_cast<size_t>(split) * routes + route) * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = acc[i];
          if constexpr (kInt8) v *= a.w2_scales[static_cast<size_t>(e) * H + h0 + (lane >> 4) * 4 + i];
          out[i] = v;
        }
      }
    }
  }
  __syncthreads();
  for (int j = static_cast<int>(threadIdx.x); j < a.num_tokens * 16; j += kSecondThreads) {
    const int t = j >> 4, c = j & 15;
    float sum = 0.0f;
    for (int k = 0; k < a.num_topk; ++k) {
      const int r = t * a.num_topk + k;
      if (ids[r] < 0) continue;
      float v = 0.0f;
      for (int s = 0; s < splits; ++s) v += y[(static_cast<size_t>(s) * routes + r) * 16 + c];
      sum = __builtin_fmaf(a.topk_weights != nullptr ? a.topk_weights[r] : 1.0f, v, sum);
    }
    const size_t o = static_cast<size_t>(t) * H + h0 + c;
    if (a.bias_0 != nullptr) sum += bf16_lo(a.bias_0[o]);
    if (a.bias_1 != nullptr) sum += bf16_lo(a.bias_1[o]);
    a.combined_x[o] = static_cast<uint16_t>(f32_to_bf16_bits(sum));
  }
}

template <bool kInt8>
hipError_t launch_few_tokens_as(const FewTokensArgs& a, hipStream_t stream) {
  const int routes = a.num_tokens * a.num_topk;
  hipLaunchKernelGGL((ep_few_tokens_gate_up_kernel<kInt8>),
                     dim3(static_cast<unsigned>(a.intermediate / 16), static_cast<unsigned>(routes)), dim3(kFirstThreads), 0,
                     stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int splits = routes >= kSecondWaves ? 1 : kSecondWaves / routes;
  const size_t lds = static_cast<size_t>(splits) * routes * 16 * sizeof(float) + routes * sizeof(int) +
                     static_cast<size_t>(routes) * (1 + kSecondWaves) * sizeof(uint16_t);
  const void* kernel = reinterpret_cast<const void*>(&ep_few_tokens_down_kernel<kInt8>);
  if (lds > 64 * 1024) {
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((ep_few_tokens_down_kernel<kInt8>), dim3(static_cast<unsigned>(a.hidden / 16)), dim3(kSecondThreads), lds,
                     stream, a, splits);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_few_tokens(const FewTokensArgs& a, hipStream_t stream) {
  if (a.num_tokens == 0) return hipSuccess;
  return a.w13_scales != nullptr ? launch_few_tokens_as<true>(a, stream) : launch_few_tokens_as<false>(a, stream);
}

}  // namespace mi_ep
