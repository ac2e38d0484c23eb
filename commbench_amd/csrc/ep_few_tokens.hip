// The whole expert layer for a few tokens in two kernels, for gfx950:
//   act[r, i] = silu(Wg[e] x[t])[i] * (Wu[e] x[t])[i]                     r = route (t, k) to expert e
//   out[t, :] = sum_k w[t, k] * W2[e_k] act[(t, k), :] (+ biases)
// With a few tokens every expert sees one or a handful of rows, so the time is that of reading the met
// experts' weights once; moving rows to the experts and back would only add launches.  Weights are
// bf16, or int8 with a scale for each output channel (widened to bf16 in registers, exactly), products
// run on the matrix units with the weights as the 16-row operand and up to 16 of an expert's routes as
// the columns, sums are fp32.  act is kept as the sum of two bf16 values (16 bits: one alone would be as large an
// error as the rounding of the result), which the second product takes as two columns.
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

// A chunk is 128 contiguous bytes of 16 weight rows, whole cache lines, in two 16-byte loads of a lane: lane l has
// row l % 16 and the l / 16-th 16 bytes of either half.  The columns' vectors are read in the same order over k, which
// is all a product needs.
template <bool kInt8>
struct Chunk {
  static constexpr int kBytes = kInt8 ? 1 : 2;
  static constexpr int kPiece = 16 / kBytes;      // elements of a load of weights
  static constexpr int kHalf = 4 * kPiece;        // of the four lanes of a row
  static constexpr int kElements = 2 * kHalf;     // of k
  static constexpr int kVectors = kInt8 ? 2 : 1;  // 16-byte bf16 loads of a column for a load of weights
  static constexpr int kAll = 2 * kVectors;       // and for a lane's whole chunk
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, kRawBufferFormat);
}
__device__ __forceinline__ void wait_lds_and_meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Who meets whom, made by every workgroup for itself from the ids: `entries` lists the met experts by their
// first routes, once for every kPass of an expert's routes (first route | pass << 10).
template <int kPass>
struct Meeting {
  uint32_t* entries;  // [routes]
  int16_t* ids;       // [routes] expert of every route, -1 for none
  int count;

  static constexpr size_t bytes(int routes) { return (static_cast<size_t>(routes) * 6 + 15) & ~static_cast<size_t>(15); }

  // scratch: num_experts words twice.  All threads; ends with the lists visible to all.
  __device__ __forceinline__ void make(const FewTokensArgs& a, int routes, unsigned char* at, int* scratch) {
    __shared__ int total;
    entries = reinterpret_cast<uint32_t*>(at);
    ids = reinterpret_cast<int16_t*>(entries + routes);
    int* first = scratch;
    int* met = scratch + a.num_experts;
    const int t = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
    for (int e = t; e < a.num_experts; e += threads) {
      first[e] = 0x7fffffff;
      met[e] = 0;
    }
    wait_lds_and_meet();
    for (int r = t; r < routes; r += threads) {
      const int64_t e = a.topk_idx[r];
      const bool routed = e >= 0 && e < a.num_experts;
      ids[r] = static_cast<int16_t>(routed ? e : -1);
      if (routed) {  // the minimum and the sum do not depend on the order of the waves
        atomicMin(first + e, r);
        atomicAdd(met + e, 1);
      }
    }
    wait_lds_and_meet();
    if (t < kWave) {
      int n = 0;
      for (int base = 0; base < routes; base += kWave) {
        const int r = base + t;
        const int e = r < routes ? ids[r] : -1;
        const int passes = e >= 0 && first[e] == r ? (met[e] + kPass - 1) / kPass : 0;
        const int upto = wave_inclusive_scan(passes);
        for (int p = 0; p < passes; ++p) entries[n + upto - passes + p] = static_cast<uint32_t>(r | p << 10);
        n += wave_read(upto, kWave - 1);
      }
      if (t == 0) total = n;
    }
    wait_lds_and_meet();
    count = __builtin_amdgcn_readfirstlane(total);
  }

  __device__ __forceinline__ int expert(int entry) const {
    return __builtin_amdgcn_readfirstlane(ids[entries[entry] & 1023]);
  }
  // An entry's routes into the wave's own list; then the lane's routes are those of columns column[c], -1 where the
  // pass has none.
  template <int kColumns>
  __device__ __forceinline__ void columns(int entry, int routes, uint16_t* list, const int (&column)[kColumns],
                                          int (&route)[kColumns]) const {
    const int lane = lane_id();
    const int packed = __builtin_amdgcn_readfirstlane(static_cast<int>(entries[entry]));
    const int e = __builtin_amdgcn_readfirstlane(ids[packed & 1023]);
    int rank = -(packed >> 10) * kPass;  // of the next match
    for (int base = packed & 1023 & ~(kWave - 1); base < routes && rank < kPass; base += kWave) {
      const bool match = base + lane < routes && ids[base + lane] == e;
      const uint64_t mask = __ballot(match);
      const int at = rank + __popcll(mask & lanes_below(lane));
      if (match && at >= 0 && at < kPass) list[at] = static_cast<uint16_t>(base + lane);
      rank += __popcll(mask);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < kColumns; ++c) route[c] = column[c] < rank ? list[column[c]] : -1;
    __builtin_amdgcn_wave_barrier();
  }
};

// The stream of chunks that a wave works through, item after item (an item: kMatrices blocks of 16 weight rows
// times the columns of an entry).  kDepth chunks are always on their way: the place of a chunk that was
// used is filled with the one kDepth further on, also across the end of an item, whose number of chunks
// is rounded up to a multiple of kDepth (the excess loads nothing).
//
// The 16 columns of a block are kFold vectors times kParts values (bf16 terms of one number) times kRoutes routes.
// kFold > 1 serves experts with few routes, where most columns would be empty: one load then fetches kFold of a
// lane's kAll vectors, vector v in the columns of fold v % kFold.  Product v has its sums in those columns of
// accumulator v % kFold; folds and parts are added up when the item ends.
template <bool kInt8, int kMatrices, int kBlocks, int kDepth, int kFold, int kParts>
struct Stream {
  using C = Chunk<kInt8>;
  static constexpr int kRoutes = 16 / (kFold * kParts);
  static constexpr int kLoads = C::kAll / kFold;
  static_assert(kLoads * kFold == C::kAll && (kFold == 1 || kBlocks == 1), "a fold fits a lane's vectors; blocks do not fold");
  vec16 w[kDepth][2][kMatrices], x[kDepth][kBlocks][kLoads];

  // Where the loads stand: an item's weights and columns, and the next chunk.
  const unsigned char* rows[kMatrices];
  int row_bytes;  // of 16 rows
  int w_lane, x_at[kBlocks], k, k_end;

  // The lane's column: route, part and fold.
  static __device__ __forceinline__ int lane_route() { return lane_id() & (kRoutes - 1); }
  static __device__ __forceinline__ int lane_part() { return (lane_id() / kRoutes) & (kParts - 1); }
  static __device__ __forceinline__ int lane_fold() { return (lane_id() & 15) / (16 / kFold); }

  __device__ __forceinline__ void load(int slot, __amdgpu_buffer_rsrc_t vectors) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool inside = k + h * C::kHalf < k_end;
      const int at = inside ? w_lane + (k + h * C::kHalf) * C::kBytes : kOutside;
#pragma unroll
      for (int m = 0; m < kMatrices; ++m)
        w[slot][h][m] = __builtin_amdgcn_raw_buffer_load_b128(rows_of(rows[m], row_bytes), at, 0, 0);
    }
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const int v = l * kFold + (kFold > 1 ? lane_fold() : 0);
      const int at = k + v / C::kVectors * C::kHalf + v % C::kVectors * 8;
      const bool inside = at < k_end;
#pragma unroll
      for (int c = 0; c < kBlocks; ++c)
        x[slot][c][l] = __builtin_amdgcn_raw_buffer_load_b128(vectors, inside ? x_at[c] + at * 2 : kOutside, 0, 0);
    }
    k += C::kElements;
  }
  __device__ __forceinline__ void use(int slot, float4v (&acc)[kMatrices][kBlocks][kFold]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < kMatrices; ++m) {
        const vec16 packed = w[slot][h][m];
        bf16x8 rows16[C::kVectors];
        if constexpr (kInt8) {
          rows16[0] = widen(packed[0], packed[1]);
          rows16[1] = widen(packed[2], packed[3]);
        } else {
          rows16[0] = as_bf16(packed);
        }
#pragma unroll
        for (int i = 0; i < C::kVectors; ++i) {
          const int v = h * C::kVectors + i;
#pragma unroll
          for (int c = 0; c < kBlocks; ++c)
            acc[m][c][v % kFold] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(rows16[i], as_bf16(x[slot][c][v / kFold]),
                                                                           acc[m][c][v % kFold], 0, 0, 0);
        }
      }
  }
  // The sums of a block, complete in the lanes of fold 0 and part 0.
  static __device__ __forceinline__ float4v total(const float4v (&acc)[kFold]) {
    float4v sum = acc[0];
    if constexpr (kFold * kParts > 1) {
      const int base = (lane_id() & 48) + lane_route();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int other = 1; other < kFold * kParts; ++other)
          sum[i] += __shfl(acc[other / kParts][i], base + other * kRoutes);
    }
    return sum;
  }
};

// Gate and up.  Items are (entry, 16 columns of act); workgroup b takes the b-th contiguous share of them.  The
// four waves split an item's k and add their sums through LDS.
template <bool kInt8, int kColumns, int kDepth>
__global__ __launch_bounds__(kFirstThreads, 4) void ep_few_tokens_gate_up_kernel(const FewTokensArgs a) {
  using C = Chunk<kInt8>;
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ float partial[2][kFirstWaves][2][4][kWave];
  __shared__ uint16_t lists[kFirstWaves][16 * kColumns];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int routes = a.num_tokens * a.num_topk;
  Meeting<16 * kColumns> meeting;
  // The experts' words lie where the sums go later: kMaxExperts words twice.
  static_assert(sizeof(partial) >= 2 * kMaxExperts * sizeof(int), "scratch of the meeting");
  meeting.make(a, routes, shared, reinterpret_cast<int*>(&partial[0][0][0][0][0]));

  const int H = a.hidden, I = a.intermediate;
  const int slices = I / 16;
  const long long items = static_cast<long long>(meeting.count) * slices;
  const long long workgroups = static_cast<long long>(gridDim.x);
  const int from = static_cast<int>(items * blockIdx.x / workgroups), to = static_cast<int>(items * (blockIdx.x + 1) / workgroups);
  if (from >= to) return;

  const int chunks = (H + C::kElements - 1) / C::kElements;
  const int share = (chunks + kFirstWaves - 1) / kFirstWaves;  // of a wave
  const int rounds = (share + kDepth - 1) / kDepth;
  const int k_lane = (lane >> 4) * C::kPiece;
  const int k_begin = share * wave * C::kElements + k_lane;
  const int share_end = share * (wave + 1) * C::kElements;
  const int k_stop = share_end < H ? share_end : H;

  const __amdgpu_buffer_rsrc_t vectors = rows_of(a.x, a.num_tokens * H * 2);
  Stream<kInt8, 2, kColumns, kDepth, 1, 1> s;
  s.row_bytes = 16 * H * C::kBytes;
  s.w_lane = (lane & 15) * H * C::kBytes;
  int column[kColumns], next_route[kColumns], route[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) column[c] = c * 16 + (lane & 15);
  int ahead = from, ahead_entry = -1;  // where the loads stand
  const auto begin_item = [&]() {
    if (ahead >= to) {
      s.k_end = 0;
      return;
    }
    const int entry = ahead / slices;
    const int e = meeting.expert(entry);
    if (entry != ahead_entry) {
      meeting.template columns<kColumns>(entry, routes, lists[wave], column, next_route);
#pragma unroll
      for (int c = 0; c < kColumns; ++c) s.x_at[c] = next_route[c] >= 0 ? next_route[c] / a.num_topk * H * 2 : kOutside;
      ahead_entry = entry;
    }
    s.rows[0] = a.w13 + (static_cast<size_t>(e) * 2 * I + (ahead - entry * slices) * 16) * H * C::kBytes;
    s.rows[1] = s.rows[0] + static_cast<size_t>(I) * H * C::kBytes;
    s.k = k_begin;
    s.k_end = k_stop;
  };
  begin_item();
#pragma unroll
  for (int d = 0; d < kDepth; ++d) s.load(d, vectors);
#pragma unroll
  for (int c = 0; c < kColumns; ++c) route[c] = next_route[c];

  for (int item = from; item < to; ++item) {
    float4v acc[2][kColumns][1];
#pragma unroll
    for (int c = 0; c < kColumns; ++c) acc[0][c][0] = acc[1][c][0] = float4v{0, 0, 0, 0};
    for (int round = 0; round < rounds; ++round) {
      if (round == rounds - 1) {
        ++ahead;
        begin_item();
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        s.use(d, acc);
        s.load(d, vectors);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int entry = item / slices;
    const int e = meeting.expert(entry), i0 = (item - entry * slices) * 16;
    // Thread 16 j + n adds up row n of column j, held by lane 16 (n / 4) + j as value n % 4.
    const int n = static_cast<int>(threadIdx.x) & 15, j = static_cast<int>(threadIdx.x) >> 4;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      float(&sums)[kFirstWaves][2][4][kWave] = partial[(item * kColumns + c) & 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sums[wave][0][i][lane] = acc[0][c][0][i];
        sums[wave][1][i][lane] = acc[1][c][0][i];
      }
      wait_lds_and_meet();
      const int column_route = __shfl(route[c], j);
      float g = 0.0f, u = 0.0f;
#pragma unroll
      for (int v = 0; v < kFirstWaves; ++v) {
        g += sums[v][0][n & 3][(n >> 2) * 16 + j];
        u += sums[v][1][n & 3][(n >> 2) * 16 + j];
      }
      if (column_route >= 0) {
        if constexpr (kInt8) {
          const float* scales = a.w13_scales + static_cast<size_t>(e) * 2 * I + i0 + n;
          g *= scales[0];
          u *= scales[I];
        }
        const float act = g / (1.0f + __expf(-g)) * u;
        const uint32_t high = f32_to_bf16_bits(act);
        uint16_t* out = a.act + static_cast<size_t>(column_route) * I + i0 + n;
        out[0] = static_cast<uint16_t>(high);
        // The rest of an infinity is none.
        const float rest = act - bf16_lo(high);
        out[static_cast<size_t>(routes) * I] = __builtin_isfinite(act) ? static_cast<uint16_t>(f32_to_bf16_bits(rest)) : 0;
      }
    }
#pragma unroll
    for (int c = 0; c < kColumns; ++c) route[c] = next_route[c];
  }
}

// Down.  Workgroup h: 16 columns of the output for every token.  Items are the entries (with fewer of them than
// waves, shares of their k); wave w takes items w, w + 8, ...  y[split][route][16] collects the products.
template <bool kInt8, int kBlocks, int kDepth, int kFold>
__global__ __launch_bounds__(kSecondThreads, 4) void ep_few_tokens_down_kernel(const FewTokensArgs a, const int splits) {
  using C = Chunk<kInt8>;
  extern __shared__ __align__(16) unsigned char shared[];
  using S = Stream<kInt8, 1, kBlocks, kDepth, kFold, 2>;
  constexpr int kPass = S::kRoutes * kBlocks;
  __shared__ uint16_t lists[kSecondWaves][kPass];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int routes = a.num_tokens * a.num_topk;
  Meeting<kPass> meeting;
  float* y = reinterpret_cast<float*>(shared + Meeting<kPass>::bytes(routes));
  meeting.make(a, routes, shared, reinterpret_cast<int*>(y));  // y's place is the scratch

  const int H = a.hidden, I = a.intermediate;
  const int h0 = static_cast<int>(blockIdx.x) * 16;
  const int items = meeting.count * splits;
  const int chunks = (I + C::kElements - 1) / C::kElements;
  const int share = (chunks + splits - 1) / splits;
  const int rounds = (share + kDepth - 1) / kDepth;
  const int k_lane = (lane >> 4) * C::kPiece;

  const __amdgpu_buffer_rsrc_t vectors = rows_of(a.act, routes * I * 4);
  S s;
  s.row_bytes = 16 * I * C::kBytes;
  s.w_lane = (lane & 15) * I * C::kBytes;
  int column[kBlocks], next_route[kBlocks], route[kBlocks];
#pragma unroll
  for (int c = 0; c < kBlocks; ++c) column[c] = c * S::kRoutes + S::lane_route();
  const int part_at = S::lane_part() * routes * I * 2;
  int ahead = wave;
  const auto begin_item = [&]() {
    if (ahead >= items) {
      s.k_end = 0;
      return;
    }
    const int entry = ahead / splits, split = ahead - entry * splits;
    meeting.template columns<kBlocks>(entry, routes, lists[wave], column, next_route);
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) s.x_at[c] = next_route[c] >= 0 ? next_route[c] * I * 2 + part_at : kOutside;
    s.rows[0] = a.w2 + (static_cast<size_t>(meeting.expert(entry)) * H + h0) * I * C::kBytes;
    const int end = share * (split + 1) * C::kElements;
    s.k = share * split * C::kElements + k_lane;
    s.k_end = end < I ? end : I;
  };
  if (wave < items) {
    begin_item();
#pragma unroll
    for (int d = 0; d < kDepth; ++d) s.load(d, vectors);
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) route[c] = next_route[c];
  }
  for (int item = wave; item < items; item += kSecondWaves) {
    float4v acc[1][kBlocks][kFold];
#pragma unroll
    for (int c = 0; c < kBlocks; ++c)
#pragma unroll
      for (int f = 0; f < kFold; ++f) acc[0][c][f] = float4v{0, 0, 0, 0};
    for (int round = 0; round < rounds; ++round) {
      if (round == rounds - 1) {
        ahead += kSecondWaves;
        begin_item();
      }
#pragma unroll
      for (int d = 0; d < kDepth; ++d) {
        s.use(d, acc);
        s.load(d, vectors);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int entry = item / splits, split = item - entry * splits;
    const int n = (lane >> 4) * 4;
    float scales[4] = {1.0f, 1.0f, 1.0f, 1.0f};
    if constexpr (kInt8) {
      const float4 of = *reinterpret_cast<const float4*>(a.w2_scales + static_cast<size_t>(meeting.expert(entry)) * H + h0 + n);
      scales[0] = of.x, scales[1] = of.y, scales[2] = of.z, scales[3] = of.w;
    }
#pragma unroll
    for (int c = 0; c < kBlocks; ++c) {
      const float4v sum = S::total(acc[0][c]);
      if (route[c] >= 0 && (lane & 15) < S::kRoutes) {
        const float4 out = {sum[0] * scales[0], sum[1] * scales[1], sum[2] * scales[2], sum[3] * scales[3]};
        *reinterpret_cast<float4*>(y + (split * routes + route[c]) * 16 + n) = out;
      }
      route[c] = next_route[c];
    }
  }
  wait_lds_and_meet();
  for (int j = static_cast<int>(threadIdx.x); j < a.num_tokens * 16; j += kSecondThreads) {
    const int t = j >> 4, c = j & 15;
    float sum = 0.0f;
    for (int k = 0; k < a.num_topk; ++k) {
      const int r = t * a.num_topk + k;
      if (meeting.ids[r] < 0) continue;
      float v = 0.0f;
      for (int split = 0; split < splits; ++split) v += y[(split * routes + r) * 16 + c];
      sum = __builtin_fmaf(a.topk_weights != nullptr ? a.topk_weights[r] : 1.0f, v, sum);
    }
    const size_t o = static_cast<size_t>(t) * H + h0 + c;
    if (a.bias_0 != nullptr) sum += bf16_lo(a.bias_0[o]);
    if (a.bias_1 != nullptr) sum += bf16_lo(a.bias_1[o]);
    a.combined_x[o] = static_cast<uint16_t>(f32_to_bf16_bits(sum));
  }
}

template <bool kInt8, int kColumns, int kDepth>
hipError_t launch_gate_up(const FewTokensArgs& a, hipStream_t stream) {
  const int routes = a.num_tokens * a.num_topk;
  DeviceTraits dev{};
  const hipError_t e = device_traits(stream, &dev);
  if (e != hipSuccess) return e;
  // As many workgroups as are resident at once, or items.
  const long long items = static_cast<long long>(routes) * (a.intermediate / 16);
  const long long resident = 4LL * dev.compute_units;
  hipLaunchKernelGGL((ep_few_tokens_gate_up_kernel<kInt8, kColumns, kDepth>),
                     dim3(static_cast<unsigned>(items < resident ? items : resident)), dim3(kFirstThreads),
                     Meeting<16 * kColumns>::bytes(routes), stream, a);
  return hipGetLastError();
}

template <bool kInt8, int kBlocks, int kDepth, int kFold>
hipError_t launch_down(const FewTokensArgs& a, hipStream_t stream) {
  const int routes = a.num_tokens * a.num_topk;
  const int splits = routes >= kSecondWaves ? 1 : kSecondWaves / routes;
  const size_t sums = static_cast<size_t>(splits) * routes * 16 * sizeof(float);
  const size_t scratch = static_cast<size_t>(a.num_experts) * 2 * sizeof(int);
  const size_t lds = Meeting<1>::bytes(routes) + (sums > scratch ? sums : scratch);
  if (lds > 60 * 1024) {
    // The kernel's LDS ceiling is raised once per device; the flags only ever go from 0 to 1.
    int ordinal = 0;
    hipError_t e = stream != nullptr ? hipStreamGetDevice(stream, &ordinal) : hipGetDevice(&ordinal);
    if (e != hipSuccess) return e;
    constexpr int kMaxDevices = 64;
    static std::atomic<int> lds_limit_raised[kMaxDevices];
    if (ordinal < 0 || ordinal >= kMaxDevices) return hipErrorInvalidDevice;
    if (lds_limit_raised[ordinal].load(std::memory_order_acquire) == 0) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(&ep_few_tokens_down_kernel<kInt8, kBlocks, kDepth, kFold>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024);
      if (e != hipSuccess) return e;
      lds_limit_raised[ordinal].store(1, std::memory_order_release);
    }
  }
  hipLaunchKernelGGL((ep_few_tokens_down_kernel<kInt8, kBlocks, kDepth, kFold>), dim3(static_cast<unsigned>(a.hidden / 16)),
                     dim3(kSecondThreads), lds, stream, a, splits);
  return hipGetLastError();
}

template <bool kInt8>
hipError_t launch_few_tokens_with(const FewTokensArgs& a, hipStream_t stream) {
  // Columns of a pass by the routes that an expert gets on average: every further pass reads its weights again.
  const int routes = a.num_tokens * a.num_topk;
  const bool many = routes > 8 * a.num_experts;
  const hipError_t e = many ? launch_gate_up<kInt8, 4, 1>(a, stream) : launch_gate_up<kInt8, 1, 2>(a, stream);
  if (e != hipSuccess) return e;
  if (many) return launch_down<kInt8, 4, 1, 1>(a, stream);
  if (routes > 2 * a.num_experts) return launch_down<kInt8, 1, 4, 1>(a, stream);
  return launch_down<kInt8, 1, 4, 2>(a, stream);
}

}  // namespace

hipError_t launch_few_tokens(const FewTokensArgs& a, hipStream_t stream) {
  if (a.num_tokens == 0) return hipSuccess;
  return a.w13_scales != nullptr ? launch_few_tokens_with<true>(a, stream) : launch_few_tokens_with<false>(a, stream);
}

}  // namespace mi_ep
