// The whole expert layer for a few tokens in two or three kernels, for gfx950:
//   act[r, i] = silu(Wg[e] x[t])[i] * (Wu[e] x[t])[i]                     r = route (t, k) to expert e
//   out[t, :] = sum_k w[t, k] * W2[e_k] act[(t, k), :] (+ biases)
// With a few tokens every expert sees one or a handful of rows, so the time is that of reading the met
// experts' weights once; moving rows to the experts and back would only add launches.  By card, 48 tokens of top 8 over 256
// experts, 7168 x 2048 int8, read 8.7 GB in 1330 to 1410 us (6.2 to 6.5 TB/s), 16 tokens over 128 experts, 4096 x 1408 bf16,
// 2.9 GB in 450 to 530 us; one token's 352 MB take 72 to 75 us, where starting and draining two kernels shows.  128 tokens of the
// first take 1890 us (11.1 GB, 5.9 TB/s).  Where experts get many routes it is far from that: 128 tokens of top 8 over 64
// experts, 4096 x 1536 int8, 587 us for 1.2 GB.  Weights are
// bf16, or int8 with a scale for each output channel (widened to bf16 in registers, exactly), products
// run on the matrix units with the weights as the 16-row operand and up to 16 of an expert's routes as
// the columns, sums are fp32.  act is kept as the sum of two bf16 values (16 bits: one alone would be as large an
// error as the rounding of the result), which the second product takes as two columns.
// A sum never depends on the order in which waves finish: each (route, output) has one writer, and the
// slots of a token are added in ascending order at the end.
#include "ep_expert.h"
#include "ep_launch.h"
#include "ep_stage.h"

namespace mi_ep {
namespace {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t words2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kFirstThreads = 256, kFirstWaves = kFirstThreads / kWave;
constexpr int kSecondThreads = 512, kSecondWaves = kSecondThreads / kWave;

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

// silu(g) * u as the sum of two bf16 values.  A finite product that bf16 would round to infinity has the largest finite
// bf16 as its first (its bits are those of the infinity less one); the rest of an infinity or a NaN is none.
__device__ __forceinline__ void activate(float g, float u, uint32_t& high, uint32_t& low) {
  const float act = g / (1.0f + __expf(-g)) * u;
  const bool finite = __builtin_isfinite(act);
  high = f32_to_bf16_bits(act);
  if (finite && (high & 0x7fffu) == 0x7f80u) --high;
  low = finite ? f32_to_bf16_bits(act - bf16_lo(high)) : 0;
}

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

// Gate and up where there are few items or many routes for an expert.  Items are (entry, 16 columns of act); workgroup b takes the b-th contiguous share of them.  The
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
        uint32_t high, low;
        activate(g, u, high, low);
        uint16_t* out = a.act + static_cast<size_t>(column_route) * I + i0 + n;
        out[0] = static_cast<uint16_t>(high);
        out[static_cast<size_t>(routes) * I] = static_cast<uint16_t>(low);
      }
    }
#pragma unroll
    for (int c = 0; c < kColumns; ++c) route[c] = next_route[c];
  }
}

// Either product where there are many (entry, 128 weight rows) items: workgroup b takes the b-th contiguous share of them.
// An item's rows are two sets of 64: the gate and the up rows of 64 columns of act, or (kDown) 128 columns of the output; wave
// w owns rows 16 w .. 16 w + 15 of each.  A stage is 128 bytes of k of the rows and the entry's vectors (kDown: both terms)
// over the same k; it comes by loads of whole lines past the registers and past the memory-side cache, which is what the
// memory delivers fastest (half a line at a time, as the products' layout has it for loads into registers, the streaming hint
// costs: 48 tokens 1850 us with it, 1560 without).  The stages of an item and of the next run on in one ring of three.
// kDown leaves y = W2[e] act as fp32 for every route; the sum over a token's slots is a kernel of its own.
constexpr int kSetRows = 64, kTileRing = 3;
constexpr int kTileVectorsAt = 2 * kSetRows * kStageK;                 // 16 vectors behind the weights, 1 KiB for four of them
template <bool kDown>
constexpr int kTileParts = kDown ? 2 : 1;
template <bool kDown>
constexpr int kTileStage = kTileVectorsAt + kTileParts<kDown> * 4 * kChunkBytes;
template <bool kDown>
constexpr int kTileScalesAt = kTileRing * kTileStage<kDown>;           // two items' scales, 256 bytes a wave
template <bool kDown>
constexpr int kTileMeetingAt = kTileScalesAt<kDown> + 2 * kFirstWaves * 256;
static_assert(kTileScalesAt<false> >= 2 * kMaxExperts * static_cast<int>(sizeof(int)), "scratch of the meeting");

template <bool kInt8, bool kDown>
__global__ __launch_bounds__(kFirstThreads, 2) void ep_few_tokens_tiles_kernel(const FewTokensArgs a) {
  constexpr int kBytes = kInt8 ? 1 : 2;
  constexpr int kElements = kStageK / kBytes;      // of k in a stage
  constexpr int kVectorBytes = 2 * kElements;      // of a column in a stage
  constexpr int kPieces = kVectorBytes / 16;       // 16 (int8 weights) or 8
  constexpr int kParts = kTileParts<kDown>, kStage = kTileStage<kDown>, kScalesAt = kTileScalesAt<kDown>;
  constexpr int kLoads = 4 + kParts, kStores = 2;  // of a wave: for a stage, for an item's results
  constexpr int kItemColumns = kDown ? 2 * kSetRows : kSetRows;
  extern __shared__ __align__(1024) unsigned char lds[];
  __shared__ uint16_t lists[kFirstWaves][16];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int routes = a.num_tokens * a.num_topk;
  Meeting<16> meeting;
  meeting.make(a, routes, lds + kTileMeetingAt<kDown>, reinterpret_cast<int*>(lds));

  const int inner = kDown ? a.intermediate : a.hidden;
  const int columns = kDown ? a.hidden : a.intermediate;          // of the result
  const int weight_rows = kDown ? a.hidden : 2 * a.intermediate;  // of an expert
  const int set_distance = kDown ? kSetRows : a.intermediate;     // rows between the two sets
  const int slices = (columns + kItemColumns - 1) / kItemColumns;
  const long long items = static_cast<long long>(meeting.count) * slices, workgroups = static_cast<long long>(gridDim.x);
  const int from = static_cast<int>(items * blockIdx.x / workgroups), to = static_cast<int>(items * (blockIdx.x + 1) / workgroups);
  if (from >= to) return;
  const int steps = (inner + kElements - 1) / kElements;
  const Place at(lane);
  const int lds_base = lds_address(lds);

  // Vectors: a load of wave w fills columns 4 w .. 4 w + 3; their pieces are permuted so that 16 lanes that read one piece of
  // the 16 columns meet all banks.  Lane l multiplies column l % 16.
  const int load_lane = lane & (4 * kPieces - 1);
  const int load_column = wave * 4 + load_lane / kPieces;
  const int load_piece = (load_lane & (kPieces - 1)) ^ (kInt8 ? load_column : load_column >> 1);
  const int read_column = lane & 15;
  const int read_vector = kTileVectorsAt + (read_column >> 2) * kChunkBytes + (read_column & 3) * kVectorBytes;
  const int column[2] = {read_column, load_column};
  const int4v desc_vectors = kDown ? descriptor_of(a.act, routes * inner * 4) : descriptor_of(a.x, a.num_tokens * inner * 2);

  int ahead = from, ahead_step = 0, ahead_entry = -1, ahead_slot = 0;  // where the loads stand
  int next_route[2] = {-1, -1}, route = -1, next_item_route = -1, vector_at = kOutside;
  int4v desc[2] = {desc_vectors, desc_vectors};
  const auto load_stage = [&]() {
    if (ahead_step == 0 && ahead < to) {
      const int entry = ahead / slices, e = meeting.expert(entry), first = (ahead - entry * slices) * kItemColumns;
      if (entry != ahead_entry) {
        meeting.template columns<2>(entry, routes, lists[wave], column, next_route);
        const int vector = kDown ? next_route[1] : next_route[1] / a.num_topk;
        vector_at = next_route[1] >= 0 && load_lane == lane ? vector * inner * 2 : kOutside;
        ahead_entry = entry;
      }
      next_item_route = next_route[0];
      const unsigned char* rows = (kDown ? a.w2 : a.w13) + (static_cast<size_t>(e) * weight_rows + first) * inner * kBytes;
#pragma unroll
      for (int set = 0; set < 2; ++set) {
        const int left = columns - first - (kDown ? set * kSetRows : 0);
        desc[set] = descriptor_of(rows + static_cast<size_t>(set * set_distance) * inner * kBytes,
                                  (left < 0 ? 0 : left < kSetRows ? left : kSetRows) * inner * kBytes);
      }
      if constexpr (kInt8) {  // lanes 0 to 15: the scales of the wave's rows of the first set, 16 to 31: of the second
        const float* scales = (kDown ? a.w2_scales : a.w13_scales) + static_cast<size_t>(e) * weight_rows;
        const int row = first + wave * 16 + (lane & 15), set = lane >> 4;
        load_word_to_lds(descriptor_of(scales, weight_rows * 4), lds_base + kScalesAt + ((ahead & 1) * kFirstWaves + wave) * 256,
                         set < 2 && row + (kDown ? set * kSetRows : 0) < columns ? (row + set * set_distance) * 4 : kOutside);
      }
    }
    const int k0 = ahead_step * kStageK;
    const int to_slot = lds_base + ahead_slot * kStage;
    const bool live = ahead < to;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int piece = at.piece_of(j);
      const int offset = live && k0 + piece < inner * kBytes ? (wave * 16 + j * 8 + at.row) * inner * kBytes + piece : kOutside;
#pragma unroll
      for (int set = 0; set < 2; ++set)
        load_to_lds<true>(desc[set], to_slot + (set * 8 + wave * 2 + j) * kChunkBytes, offset, k0);
    }
    const int k = ahead_step * kVectorBytes;
    const int offset = live && vector_at >= 0 && k + load_piece * 16 < inner * 2 ? vector_at + load_piece * 16 : kOutside;
#pragma unroll
    for (int part = 0; part < kParts; ++part)
      load_to_lds(desc_vectors, to_slot + kTileVectorsAt + (part * 4 + wave) * kChunkBytes, offset, k + part * routes * inner * 2);
    ahead_slot = ahead_slot + 1 == kTileRing ? 0 : ahead_slot + 1;
    if (++ahead_step == steps) {
      ahead_step = 0;
      ++ahead;
    }
  };
  const __amdgpu_buffer_rsrc_t result = kDown ? rows_of(a.y, routes * columns * 4) : rows_of(a.act, routes * columns * 4);

#pragma unroll
  for (int s = 0; s < kTileRing - 1; ++s) load_stage();
  int slot = 0, since = kTileRing;  // stages since the last results were stored
  for (int item = from; item < to; ++item) {
    // At the start of an item the loads are two stages ahead, still in this item: it has two stages at least.
    float4v sum[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    for (int step = 0; step < steps; ++step) {
      // This stage is in (the next one and an item's stores may be on their way), and every wave has left the stage before
      // it, whose place the next load takes.
      if (since < kTileRing - 1)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((kTileRing - 2) * kLoads + kStores) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((kTileRing - 2) * kLoads) : "memory");
      ++since;
      if (step == 0) route = next_item_route;
      load_stage();
      const unsigned char* stage = lds + slot * kStage;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // Rows are permuted by half their number, as Place says.
        const int group = h * 4 + (lane >> 4), piece = (group ^ ((read_column >> 1) & 7)) * 16;
        vec16 w[2];
#pragma unroll
        for (int set = 0; set < 2; ++set)
          w[set] = *reinterpret_cast<const vec16*>(stage + (set * kSetRows + wave * 16 + read_column) * kStageK + piece);
#pragma unroll
        for (int i = 0; i < (kInt8 ? 2 : 1); ++i) {
          const int of = kInt8 ? ((group * 2 + i) ^ read_column) * 16 : (group ^ (read_column >> 1)) * 16;
          bf16x8 rows[2];
#pragma unroll
          for (int set = 0; set < 2; ++set) rows[set] = kInt8 ? widen(w[set][2 * i], w[set][2 * i + 1]) : as_bf16(w[set]);
#pragma unroll
          for (int part = 0; part < kParts; ++part) {
            const bf16x8 x = as_bf16(*reinterpret_cast<const vec16*>(stage + read_vector + part * 4 * kChunkBytes + of));
#pragma unroll
            for (int set = 0; set < 2; ++set) sum[set] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(rows[set], x, sum[set], 0, 0, 0);
          }
        }
      }
      slot = slot + 1 == kTileRing ? 0 : slot + 1;
    }
    // Lane l holds rows 4 (l / 16) + 0..3 of column l % 16.
    const int first = item % slices * kItemColumns + wave * 16 + (lane >> 4) * 4;
    if constexpr (kInt8) {
      const float* scales = reinterpret_cast<const float*>(lds + kScalesAt + ((item & 1) * kFirstWaves + wave) * 256);
#pragma unroll
      for (int set = 0; set < 2; ++set) {
        const float4 of = *reinterpret_cast<const float4*>(scales + set * 16 + (lane >> 4) * 4);
        sum[set][0] *= of.x, sum[set][1] *= of.y, sum[set][2] *= of.z, sum[set][3] *= of.w;
      }
    }
    if constexpr (kDown) {
#pragma unroll
      for (int set = 0; set < 2; ++set) {
        const int c = first + set * kSetRows;
        const vec16 bits = {__float_as_uint(sum[set][0]), __float_as_uint(sum[set][1]), __float_as_uint(sum[set][2]),
                            __float_as_uint(sum[set][3])};
        __builtin_amdgcn_raw_buffer_store_b128(bits, result, route >= 0 && c < columns ? (route * columns + c) * 4 : kOutside, 0,
                                               kCachePolicyDeviceScope);
      }
    } else {
      uint32_t high[4], low[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) activate(sum[0][i], sum[1][i], high[i], low[i]);
      const int offset = route >= 0 && first < columns ? (route * columns + first) * 2 : kOutside;
      __builtin_amdgcn_raw_buffer_store_b64(words2{high[0] | high[1] << 16, high[2] | high[3] << 16}, result, offset, 0,
                                            kCachePolicyDeviceScope);
      __builtin_amdgcn_raw_buffer_store_b64(words2{low[0] | low[1] << 16, low[2] | low[3] << 16}, result, offset,
                                            routes * columns * 2, kCachePolicyDeviceScope);
    }
    since = 0;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load outlives the workgroup's LDS
}

// out[t] = sum_k w[t, k] y[(t, k)] + biases, the slots in ascending order; a thread four columns.
__global__ __launch_bounds__(kFirstThreads) void ep_few_tokens_sum_kernel(const FewTokensArgs a) {
  const int quads = a.hidden / 4;
  const int index = static_cast<int>(blockIdx.x) * kFirstThreads + static_cast<int>(threadIdx.x);
  const int t = index / quads, c = (index - t * quads) * 4;
  if (t >= a.num_tokens) return;
  float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int k = 0; k < a.num_topk; ++k) {
    const int r = t * a.num_topk + k;
    const int64_t e = a.topk_idx[r];
    if (e < 0 || e >= a.num_experts) continue;
    const float w = a.topk_weights != nullptr ? a.topk_weights[r] : 1.0f;
    const float4 v = *reinterpret_cast<const float4*>(a.y + static_cast<size_t>(r) * a.hidden + c);
    sum[0] = __builtin_fmaf(w, v.x, sum[0]), sum[1] = __builtin_fmaf(w, v.y, sum[1]);
    sum[2] = __builtin_fmaf(w, v.z, sum[2]), sum[3] = __builtin_fmaf(w, v.w, sum[3]);
  }
  const size_t o = static_cast<size_t>(t) * a.hidden + c;
  for (const uint16_t* bias : {a.bias_0, a.bias_1})
    if (bias != nullptr)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += bf16_lo(bias[o + i]);
  *reinterpret_cast<uint2*>(a.combined_x + o) = uint2{to_bf16_pair(sum[0], sum[1]), to_bf16_pair(sum[2], sum[3])};
}

// Down where there are few items, or many routes for an expert.  Workgroup h: 16 columns of the output for every token.  Items are the entries (with fewer of them than
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

template <bool kInt8, bool kDown>
hipError_t launch_tiles(const FewTokensArgs& a, int compute_units, hipStream_t stream) {
  const int lds = kTileMeetingAt<kDown> + static_cast<int>(Meeting<16>::bytes(a.num_tokens * a.num_topk));
  static LdsCeiling ceiling;
  const hipError_t e =
      ceiling.raise(reinterpret_cast<const void*>(&ep_few_tokens_tiles_kernel<kInt8, kDown>), 96 * 1024, stream);
  if (e != hipSuccess) return e;
  // Two workgroups a compute unit; the second product's have room for each other up to 853 routes.  Beyond, the grid's second half
  // follows the first (106 tokens of top 8 over 256 experts, 7168 x 2048, 1768 us, 107 tokens 1869).
  hipLaunchKernelGGL((ep_few_tokens_tiles_kernel<kInt8, kDown>), dim3(static_cast<unsigned>(2 * compute_units)),
                     dim3(kFirstThreads), lds, stream, a);
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
    static LdsCeiling ceiling;
    const hipError_t e =
        ceiling.raise(reinterpret_cast<const void*>(&ep_few_tokens_down_kernel<kInt8, kBlocks, kDepth, kFold>), 80 * 1024, stream);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((ep_few_tokens_down_kernel<kInt8, kBlocks, kDepth, kFold>), dim3(static_cast<unsigned>(a.hidden / 16)),
                     dim3(kSecondThreads), lds, stream, a, splits);
  return hipGetLastError();
}

template <bool kInt8>
hipError_t launch_few_tokens_with(const FewTokensArgs& a, hipStream_t stream) {
  // Columns of a pass by the routes that an expert gets on average: every further pass reads its weights again.  Four
  // blocks of 16 columns leave no registers for loads further ahead (with int8 weights 32 are spilled): 128 tokens of top 8
  // over 64 experts, 4096 x 1536, read their weights at 2 TB/s.
  const int routes = a.num_tokens * a.num_topk;
  const bool many = routes > 8 * a.num_experts;
  DeviceTraits dev{};
  hipError_t e = device_traits(stream, &dev);
  if (e != hipSuccess) return e;
  // Tiles where every workgroup gets two items or more, on (at most) so many experts.  Without / with tiles in us: 48 tokens
  // of top 8 over 256 experts, 7168 x 2048 int8 1564 / 1412; 16 over 128, 4096 x 1408 bf16 580 / 531; 4 tokens of the first
  // (1024 items) 271 / 243, one token (256) 76 / 81; 12 tokens of top 4 over 64 experts, 4096 x 1024 (768) 116 / 128.
  const long long met = routes < a.num_experts ? routes : a.num_experts;
  const auto tiles = [&](int inner, int columns, int item_columns, int items_for_unit) {
    const long long items = met * ((columns + item_columns - 1) / item_columns);
    return !many && inner > kStageK && items >= static_cast<long long>(items_for_unit) * dev.compute_units;
  };
  e = many ? launch_gate_up<kInt8, 4, 1>(a, stream)
      : tiles(a.hidden, a.intermediate, kSetRows, 4) ? launch_tiles<kInt8, false>(a, dev.compute_units, stream)
                                                  : launch_gate_up<kInt8, 1, 2>(a, stream);
  if (e != hipSuccess) return e;
  // The second product's tiles cost a launch and the traffic of y, and pay by the items: 48 tokens (14336 items) 1407 / 1329,
  // 16 tokens (4096) 529 / 531, which is where they begin to, 12 tokens (1536) 115 / 122.
  if (tiles(a.intermediate, a.hidden, 2 * kSetRows, 16)) {
    e = launch_tiles<kInt8, true>(a, dev.compute_units, stream);
    if (e != hipSuccess) return e;
    const long long threads = static_cast<long long>(a.num_tokens) * (a.hidden / 4);
    hipLaunchKernelGGL(ep_few_tokens_sum_kernel, dim3(static_cast<unsigned>((threads + kFirstThreads - 1) / kFirstThreads)),
                       dim3(kFirstThreads), 0, stream, a);
    return hipGetLastError();
  }
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
