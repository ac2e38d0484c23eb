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
#include <atomic>

#include "ep_device.h"

namespace mi_ep {
namespace {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kFirstThreads = 256, kFirstWaves = kFirstThreads / kWave;
constexpr int kSecondThreads = 512, kSecondWaves = kSecondThreads / kWave;
constexpr int kOutside = static_cast<int>(0x80000000u);  // an offset beyond every descriptor: the load returns zeros

// 8 of the int8 codes in two words as bf16 (every code is one exactly).
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  uint32_t f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t word = j < 4 ? lo : hi;
    f[j] = __float_as_uint(static_cast<float>(static_cast<int8_t>(word >> (8 * (j & 3)))));
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

// A chunk is what 64 lanes take of 16 weight rows in one 16-byte load each: lane l has row l % 16 and the l / 16-th
// piece of 64 contiguous bytes.  The columns' vectors are read in the same order over k, which is all a
// product needs.
template <bool kInt8>
struct Chunk {
  static constexpr int kBytes = kInt8 ? 1 : 2;
  static constexpr int kLane = 16 / kBytes;      // elements of a lane
  static constexpr int kElements = 4 * kLane;    // of k
  static constexpr int kVectors = kInt8 ? 2 : 1; // 16-byte bf16 loads of a column for them
};

// acc[m][c] += W[m][16 rows] . X[16 columns of c] over chunks [begin, end) of k: kBatch chunks of weights and
// columns are loaded before the first product, so that many bytes are on their way whatever the latency.  w_at, x_at:
// the lane's byte offsets at k = 0; a lane without a column has kOutside.
template <bool kInt8, int kMatrices, int kColumns, int kBatch>
__device__ __forceinline__ void multiply(const __amdgpu_buffer_rsrc_t (&w)[kMatrices], int w_at, __amdgpu_buffer_rsrc_t x,
                                         const int (&x_at)[kColumns], int begin, int end, int length,
                                         float4v (&acc)[kMatrices][kColumns]) {
  using C = Chunk<kInt8>;
  const int k_lane = (lane_id() >> 4) * C::kLane;
  for (int chunk = begin; chunk < end; chunk += kBatch) {
    vec16 wv[kBatch][kMatrices], xv[kBatch][kColumns][C::kVectors];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      // Chunks behind the range, and the lanes of the last one behind the row, read nothing.
      const bool inside = chunk + b < end && (chunk + b) * C::kElements + k_lane < length;
      const int at = inside ? w_at + (chunk + b) * 64 : kOutside;
#pragma unroll
      for (int m = 0; m < kMatrices; ++m) wv[b][m] = __builtin_amdgcn_raw_buffer_load_b128(w[m], at, 0, kCachePolicyStreaming);
#pragma unroll
      for (int c = 0; c < kColumns; ++c) {
        const int from = inside ? x_at[c] + (chunk + b) * C::kElements * 2 : kOutside;
#pragma unroll
        for (int v = 0; v < C::kVectors; ++v) xv[b][c][v] = __builtin_amdgcn_raw_buffer_load_b128(x, from + 16 * v, 0, 0);
      }
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int m = 0; m < kMatrices; ++m) {
        if constexpr (kInt8) {
          const bf16x8 w0 = widen(wv[b][m][0], wv[b][m][1]), w1 = widen(wv[b][m][2], wv[b][m][3]);
#pragma unroll
          for (int c = 0; c < kColumns; ++c) {
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, as_bf16(xv[b][c][0]), acc[m][c], 0, 0, 0);
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, as_bf16(xv[b][c][C::kVectors - 1]), acc[m][c], 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kColumns; ++c)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16(wv[b][m]), as_bf16(xv[b][c][0]), acc[m][c], 0, 0, 0);
        }
      }
  }
}

__device__ __forceinline__ int expert_of(const FewTokensArgs& a, int route, int routes) {
  if (route >= routes) return -1;
  const int64_t e = a.topk_idx[route];
  return e >= 0 && e < a.num_experts ? static_cast<int>(e) : -1;
}

// The routes of expert e in order into a wave's own list; returns how many.  The ids come from LDS or memory.
template <typename Ids>
__device__ __forceinline__ int collect_routes(const Ids& ids, int routes, int e, uint16_t* list) {
  const int lane = lane_id();
  int n = 0;
  for (int base = 0; base < routes; base += kWave) {
    const bool match = ids(base + lane) == e;
    const uint64_t mask = __ballot(match);
    if (match) list[n + __popcll(mask & lanes_below(lane))] = static_cast<uint16_t>(base + lane);
    n += __popcll(mask);
  }
  __builtin_amdgcn_wave_barrier();
  return n;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, kRawBufferFormat);
}

// kColumns blocks of 16 routes from c0 on, through 16 gate and 16 up rows: the waves share out k.
template <bool kInt8, int kColumns, int kBatch>
__device__ __forceinline__ void gate_up(const FewTokensArgs& a, int e, int i0, const uint16_t* list, int count, int c0,
                                        float (&partial)[kFirstWaves][2][4][kWave]) {
  using C = Chunk<kInt8>;
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  const int H = a.hidden, I = a.intermediate;
  const unsigned char* gate = a.w13 + (static_cast<size_t>(e) * 2 * I + i0) * H * C::kBytes;
  const __amdgpu_buffer_rsrc_t w[2] = {rows_of(gate, 16 * H * C::kBytes),
                                       rows_of(gate + static_cast<size_t>(I) * H * C::kBytes, 16 * H * C::kBytes)};
  int x_at[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    const int column = c0 + c * 16 + (lane & 15);
    x_at[c] = column < count ? list[column] / a.num_topk * H * 2 + (lane >> 4) * C::kLane * 2 : kOutside;
  }
  float4v acc[2][kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) acc[0][c] = acc[1][c] = float4v{0, 0, 0, 0};
  const int chunks = (H + C::kElements - 1) / C::kElements;
  multiply<kInt8, 2, kColumns, kBatch>(w, (lane & 15) * H * C::kBytes + (lane >> 4) * 16, rows_of(a.x, a.num_tokens * H * 2),
                                       x_at, chunks * wave / kFirstWaves, chunks * (wave + 1) / kFirstWaves, H, acc);
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    if (c0 + c * 16 >= count) break;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      partial[wave][0][i][lane] = acc[0][c][i];
      partial[wave][1][i][lane] = acc[1][c][i];
    }
    __syncthreads();
    // Thread 16 j + n: row n of column j, held by lane 16 (n / 4) + j as value n % 4.
    const int n = static_cast<int>(threadIdx.x) & 15, j = static_cast<int>(threadIdx.x) >> 4;
    const int column = c0 + c * 16 + j;
    if (column < count) {
      float g = 0.0f, u = 0.0f;
#pragma unroll
      for (int v = 0; v < kFirstWaves; ++v) {
        g += partial[v][0][n & 3][(n >> 2) * 16 + j];
        u += partial[v][1][n & 3][(n >> 2) * 16 + j];
      }
      if constexpr (kInt8) {
        const float* scales = a.w13_scales + static_cast<size_t>(e) * 2 * I + i0 + n;
        g *= scales[0];
        u *= scales[I];
      }
      a.act[static_cast<size_t>(list[column]) * I + i0 + n] =
          static_cast<uint16_t>(f32_to_bf16_bits(g / (1.0f + __expf(-g)) * u));
    }
  }
}

// Workgroup (s, r): 16 columns of act for the expert of route r, if r is that expert's first route.
template <bool kInt8>
__global__ __launch_bounds__(kFirstThreads, 4) void ep_few_tokens_gate_up_kernel(const FewTokensArgs a) {
  __shared__ uint16_t lists[kFirstWaves][kFewRoutes];
  __shared__ float partial[kFirstWaves][2][4][kWave];
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int routes = a.num_tokens * a.num_topk;
  const int r = static_cast<int>(blockIdx.y);
  const int e = expert_of(a, r, routes);
  uint16_t* list = lists[wave];  // every wave makes its own: no barrier before the first load
  const int count = e < 0 ? 0 : collect_routes([&](int q) { return expert_of(a, q, routes); }, routes, e, list);
  const bool leads = count > 0 && list[0] == r;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.leaders[r] = leads ? 1 : 0;
  if (!leads) return;
  const int i0 = static_cast<int>(blockIdx.x) * 16;
  for (int c0 = 0; c0 < count;) {
    const int left = count - c0;
    if (left <= 16) {
      gate_up<kInt8, 1, 4>(a, e, i0, list, count, c0, partial);
      c0 += 16;
    } else if (left <= 32) {
      gate_up<kInt8, 2, 2>(a, e, i0, list, count, c0, partial);
      c0 += 32;
    } else {
      gate_up<kInt8, 4, 1>(a, e, i0, list, count, c0, partial);
      c0 += 64;
    }
  }
}

// kColumns blocks of 16 routes from c0 on, through 16 rows of the down weights over chunks [begin, end).
template <bool kInt8, int kColumns, int kBatch>
__device__ __forceinline__ void down(const FewTokensArgs& a, int e, int h0, const uint16_t* list, int count, int c0, int begin,
                                     int end, float* y) {
  using C = Chunk<kInt8>;
  const int lane = lane_id();
  const int H = a.hidden, I = a.intermediate;
  const __amdgpu_buffer_rsrc_t w[1] = {rows_of(a.w2 + (static_cast<size_t>(e) * H + h0) * I * C::kBytes, 16 * I * C::kBytes)};
  int x_at[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    const int column = c0 + c * 16 + (lane & 15);
    x_at[c] = column < count ? list[column] * I * 2 + (lane >> 4) * C::kLane * 2 : kOutside;
  }
  float4v acc[1][kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) acc[0][c] = float4v{0, 0, 0, 0};
  multiply<kInt8, 1, kColumns, kBatch>(w, (lane & 15) * I * C::kBytes + (lane >> 4) * 16,
                                       rows_of(a.act, a.num_tokens * a.num_topk * I * 2), x_at, begin, end, I, acc);
  float scales[4] = {1.0f, 1.0f, 1.0f, 1.0f};
  if constexpr (kInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) scales[i] = a.w2_scales[static_cast<size_t>(e) * H + h0 + (lane >> 4) * 4 + i];
  }
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    const int column = c0 + c * 16 + (lane & 15);
    if (column < count) {
      float* out = y + list[column] * 16 + (lane >> 4) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = acc[0][c][i] * scales[i];
    }
  }
}

// Workgroup h: 16 columns of the output for every token.  The waves share out the met experts (and, with
// fewer experts than waves, ranges of the intermediate axis); y[split][route][16] collects their products.
template <bool kInt8>
__global__ __launch_bounds__(kSecondThreads, 4) void ep_few_tokens_down_kernel(const FewTokensArgs a, const int splits) {
  extern __shared__ float y[];
  const int routes = a.num_tokens * a.num_topk;
  int* ids = reinterpret_cast<int*>(y + splits * routes * 16);
  uint16_t* leaders = reinterpret_cast<uint16_t*>(ids + routes);
  uint16_t* lists = leaders + routes;  // [kSecondWaves][routes]
  __shared__ int met;
  const int lane = lane_id(), wave = static_cast<int>(threadIdx.x) >> 6;
  for (int r = static_cast<int>(threadIdx.x); r < routes; r += kSecondThreads) ids[r] = expert_of(a, r, routes);
  if (wave == kSecondWaves - 1) {  // the first route of every met expert, in order
    const int n = collect_routes([&](int r) { return r < routes ? a.leaders[r] : 0; }, routes, 1, leaders);
    if (lane == 0) met = n;
  }
  __syncthreads();

  const int h0 = static_cast<int>(blockIdx.x) * 16;
  const int chunks = (a.intermediate + Chunk<kInt8>::kElements - 1) / Chunk<kInt8>::kElements;
  uint16_t* list = lists + wave * routes;
  for (int item = wave; item < met * splits; item += kSecondWaves) {
    const int leader = item / splits, split = item - leader * splits;
    const int e = ids[leaders[leader]];
    const int count = collect_routes([&](int r) { return r < routes ? ids[r] : -1; }, routes, e, list);
    const int begin = chunks * split / splits, end = chunks * (split + 1) / splits;
    float* to = y + split * routes * 16;
    for (int c0 = 0; c0 < count;) {
      const int left = count - c0;
      if (left <= 16) {
        down<kInt8, 1, 8>(a, e, h0, list, count, c0, begin, end, to);
        c0 += 16;
      } else if (left <= 32) {
        down<kInt8, 2, 4>(a, e, h0, list, count, c0, begin, end, to);
        c0 += 32;
      } else {
        down<kInt8, 4, 2>(a, e, h0, list, count, c0, begin, end, to);
        c0 += 64;
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
      for (int s = 0; s < splits; ++s) v += y[(s * routes + r) * 16 + c];
      sum = __builtin_fmaf(a.topk_weights != nullptr ? a.topk_weights[r] : 1.0f, v, sum);
    }
    const size_t o = static_cast<size_t>(t) * a.hidden + h0 + c;
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
  if (lds > 64 * 1024) {
    // The kernel's LDS ceiling is raised once per device; the flags only ever go from 0 to 1.
    int ordinal = 0;
    e = stream != nullptr ? hipStreamGetDevice(stream, &ordinal) : hipGetDevice(&ordinal);
    if (e != hipSuccess) return e;
    constexpr int kMaxDevices = 64;
    static std::atomic<int> lds_limit_raised[kMaxDevices];
    if (ordinal < 0 || ordinal >= kMaxDevices) return hipErrorInvalidDevice;
    if (lds_limit_raised[ordinal].load(std::memory_order_acquire) == 0) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(&ep_few_tokens_down_kernel<kInt8>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024);
      if (e != hipSuccess) return e;
      lds_limit_raised[ordinal].store(1, std::memory_order_release);
    }
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
