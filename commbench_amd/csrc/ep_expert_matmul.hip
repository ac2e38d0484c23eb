// The experts' products on dispatched rows, int8 x int8 with a scale for each row and each output
// channel, for gfx950:
//   c[m, n] = a_scale[m] * b_scale[e, n] * sum_k a[m, k] * b[e, n, k]     rows m of expert e's segment
//   out = bf16(c)   or, gate and up in one product,   out[m, i] = bf16(silu(c[m, i]) * c[m, I + i])
// The sum over k is exact in 32-bit integers (|a|, |b| <= 128 and k < 2^17); the scales, silu and the product are fp32,
// rounded to bf16 once.  silu(gate) * up is formed where both sums lie in one lane, so the 2 I columns never reach memory.
//
// What bounds it depends on the rows of an expert.  Few rows: reading the weights once (256 experts x 4096 x 7168 with 2 rows
// each 1071 us, 7.0 TB/s; with 32 rows 1126).  Hundreds: the matrix units at the clock that the card's power limit leaves
// them (8192^3 442 to 474 us by card, 2490 to 2320 TOP/s, clock near 1.6 GHz), less what ragged heights leave empty: a segment is
// computed in blocks of 64 rows (8192 tokens' 65536 rows over 256 experts x 4096 x 7168: 2390 to 2450 us, of which the empty
// part of the blocks is an eighth; the matrix units are busy for 46 % of it at 1.8 GHz, since weights that nobody has read
// before are asked for about one stage, 1 us, ahead).
#include <type_traits>

#include "ep_expert.h"
#include "ep_launch.h"
#include "ep_stage.h"

namespace mi_ep {
namespace {

typedef int int16v __attribute__((ext_vector_type(16)));
typedef uint32_t words2 __attribute__((ext_vector_type(2)));

struct Segment {
  int first, rows;
};
__device__ __forceinline__ Segment segment_of(const ExpertMatmulArgs& a, int e) {
  long long lo = 0, hi = a.num_rows;
  if (a.expert_offsets != nullptr) {
    lo = a.expert_offsets[e];
    hi = a.num_tokens_per_expert != nullptr ? lo + a.num_tokens_per_expert[e] : a.expert_offsets[e + 1];
  }
  if (lo < 0) lo = 0;
  if (hi > a.num_rows) hi = a.num_rows;
  return hi > lo ? Segment{static_cast<int>(lo), static_cast<int>(hi - lo)} : Segment{0, 0};
}

// v / (1 + exp(-v)); the reciprocal instruction is off by one unit in the last place at most.
__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.0f + __expf(-v)); }

// ---- small tiles: 64 rows by 64 columns, for problems of few tiles or of a few rows an expert -------------
// A workgroup a tile, so that little work still spreads over the card (8 experts x 32 rows x 512 x 256: 5.4 us) and two or
// three workgroups of a compute unit hide one another's start; a ring of three stages each.
constexpr int kTileM = 64, kTileN = 64;
constexpr int kSmallThreads = 256;

struct RowTile {
  int expert, first, rows;  // rows [first, first + rows) of a and out; rows == 0: no such tile
  int only;                 // no other tile has rows of the expert
};

// The `index`-th tile of up to kTileM rows, the experts' segments cut into tiles one after the other.
__device__ __forceinline__ RowTile find_row_tile(const ExpertMatmulArgs& a, int index) {
  if (a.expert_offsets == nullptr) {
    const int left = a.num_rows - index * kTileM;
    return RowTile{0, index * kTileM, left < 0 ? 0 : left < kTileM ? left : kTileM, a.num_rows <= kTileM ? 1 : 0};
  }
  __shared__ int wave_tiles[kSmallThreads / kWave];
  __shared__ RowTile found;
  const int t = static_cast<int>(threadIdx.x);
  const int per = (a.num_experts + kSmallThreads - 1) / kSmallThreads;
  if (t == 0) found = RowTile{0, 0, 0, 0};
  Segment segments[kMaxExperts / kSmallThreads];
  int mine = 0;
#pragma unroll
  for (int j = 0; j < kMaxExperts / kSmallThreads; ++j) {
    const int e = t * per + j;
    segments[j] = j < per && e < a.num_experts ? segment_of(a, e) : Segment{0, 0};
    mine += (segments[j].rows + kTileM - 1) / kTileM;
  }
  const int upto = wave_inclusive_scan(mine);
  if (lane_id() == kWave - 1) wave_tiles[t >> 6] = upto;
  __syncthreads();
  int before = upto - mine;
  for (int w = 0; w < (t >> 6); ++w) before += wave_tiles[w];
#pragma unroll
  for (int j = 0; j < kMaxExperts / kSmallThreads; ++j) {
    const int tiles = (segments[j].rows + kTileM - 1) / kTileM;
    if (index >= before && index < before + tiles) {
      const int skip = (index - before) * kTileM;
      found = RowTile{t * per + j, segments[j].first + skip,
                      segments[j].rows - skip < kTileM ? segments[j].rows - skip : kTileM, tiles == 1 ? 1 : 0};
    }
    before += tiles;
  }
  __syncthreads();
  return RowTile{__builtin_amdgcn_readfirstlane(found.expert), __builtin_amdgcn_readfirstlane(found.first),
                 __builtin_amdgcn_readfirstlane(found.rows), __builtin_amdgcn_readfirstlane(found.only)};
}

// Wave (mw, nw) owns 32 rows and 32 columns (with kSilu their gate and their up channels).
template <bool kSilu>
__global__ __launch_bounds__(kSmallThreads) void ep_expert_matmul_small_kernel(const ExpertMatmulArgs a) {
  constexpr int kSets = kSilu ? 2 : 1;
  constexpr int kRing = 3;
  constexpr int kABytes = kTileM * kStageK, kStage = kABytes + kSets * kTileN * kStageK;
  constexpr int kLoads = 2 * (1 + kSets);  // of a wave for a stage
  __shared__ __align__(1024) unsigned char ring[kRing * kStage];
  const RowTile tile = find_row_tile(a, static_cast<int>(blockIdx.y));
  if (tile.rows <= 0) return;
  const int K = a.in_features;
  const int columns = kSilu ? a.out_features / 2 : a.out_features;
  const int n0 = static_cast<int>(blockIdx.x) * kTileN;
  const int lane = lane_id(), r = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int mw = wave & 1, nw = wave >> 1;
  const int steps = (K + kStageK - 1) / kStageK;
  const Place at(lane);
  const int b_rows = columns - n0 < kTileN ? columns - n0 : kTileN;
  const size_t channel = static_cast<size_t>(tile.expert) * a.out_features + n0;
  const int4v desc_a = descriptor_of(a.a + static_cast<size_t>(tile.first) * K, tile.rows * K);
  const int4v desc_b = descriptor_of(a.b + channel * K, b_rows * K);
  const int4v desc_up = kSilu ? descriptor_of(a.b + (channel + columns) * K, b_rows * K) : desc_b;
  const int offset = (wave * 16 + at.row) * K;
  const int ring_base = lds_address(ring);
  int16v acc[kSets];
#pragma unroll
  for (int s = 0; s < kSets; ++s) acc[s] = int16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  const auto products = [&](auto once) {
    constexpr bool kOnce = decltype(once)::value;
    int load_slot = 0;
    const auto load_stage = [&](int step) {  // steps behind the last load nothing, but count
      const int k0 = step < steps ? step * kStageK : 0;
      const int to = ring_base + load_slot * kStage + wave * 2 * kChunkBytes;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int piece = at.piece_of(j);
        const int from = step * kStageK + piece < K ? offset + j * 8 * K + piece : kOutside;
        load_to_lds(desc_a, to + j * kChunkBytes, from, k0);
        load_to_lds<kOnce>(desc_b, to + kABytes + j * kChunkBytes, from, k0);
        if constexpr (kSilu) load_to_lds<kOnce>(desc_up, to + kABytes + kTileN * kStageK + j * kChunkBytes, from, k0);
      }
      load_slot = load_slot + 1 == kRing ? 0 : load_slot + 1;
    };
#pragma unroll
    for (int s = 0; s < kRing - 1; ++s) load_stage(s);
    int slot = 0;
    for (int step = 0; step < steps; ++step) {
      // Stage step is in, and every wave has left the stage before it, whose place the next load takes.
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"((kRing - 2) * kLoads) : "memory");
      load_stage(step + kRing - 1);
      const unsigned char* stage = ring + slot * kStage;
#pragma unroll
      for (int quarter = 0; quarter < 4; ++quarter) {
        const unsigned char* base = stage + (at.read_at ^ (quarter * 32));
        const int4v rows = *reinterpret_cast<const int4v*>(base + mw * 32 * kStageK);
#pragma unroll
        for (int s = 0; s < kSets; ++s) {
          const int4v channels = *reinterpret_cast<const int4v*>(base + kABytes + (s * kTileN + nw * 32) * kStageK);
          acc[s] = __builtin_amdgcn_mfma_i32_32x32x32_i8(channels, rows, acc[s], 0, 0, 0);
        }
      }
      slot = slot + 1 == kRing ? 0 : slot + 1;
    }
  };
  if (tile.only != 0) products(std::true_type{});
  else products(std::false_type{});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load outlives the workgroup's LDS

  // Lane l holds row l % 32 and channels 8 g + 4 (l / 32) + 0..3.
  const int row = mw * 32 + r;
  if (row >= tile.rows) return;
  const float row_scale = a.a_scales[static_cast<size_t>(tile.first + row) * a.a_scales_row_stride];
  const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(a.out + static_cast<size_t>(tile.first) * columns, 0,
                                                                       tile.rows * columns * 2, kRawBufferFormat);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + nw * 32 + g * 8 + (lane >> 5) * 4;
    if (n >= columns) break;
    const float* scales = a.b_scales + static_cast<size_t>(tile.expert) * a.out_features + n;
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = static_cast<float>(acc[0][g * 4 + i]) * (row_scale * scales[i]);
      if constexpr (kSilu) o[i] = silu(o[i]) * (static_cast<float>(acc[kSets - 1][g * 4 + i]) * (row_scale * scales[columns + i]));
    }
    __builtin_amdgcn_raw_buffer_store_b64(words2{to_bf16_pair(o[0], o[1]), to_bf16_pair(o[2], o[3])}, out,
                                          (row * columns + n) * 2, 0, kCachePolicyDeviceScope);
  }
}

// ---- large tiles: up to 256 rows by 256 channels ----------------------------------------------------------
// One persistent workgroup a compute unit, four waves of 128 x 128: a stage's 64 KiB give 128 products of 32 x 32 x 32, half
// a fragment read from LDS for each, and the accumulators fill the 256 registers that the products can add to directly.
// The rest does not quite fit: 4 vector registers and 178 (silu 243) scalar ones are spilled.
// With loads of 128 bytes a row (64: a sixth slower), LDS rows permuted so that no bank is met twice, reads and loads spread
// between the products one by one, and the next tile's loads and this tile's stores on their way at once.
// Rejected: 320-row tiles (the accumulators no longer fit beside the fragments and are copied about), tiles claimed from
// counters (skewed routing 4 % slower, even routing 2 % faster), dies' runs cut by cost instead of by tiles (no gain).
constexpr int kBigN = 256;       // channels of a tile: with kSilu 128 gate channels and their 128 up channels
constexpr int kBlockRows = 64;   // a tile's rows come in pairs of 32-row blocks, one for each half of the waves
constexpr int kMaxBlocks = 4;    // 256 rows: the accumulators fill the matrix units' own registers
// With silu 257 to 320 rows make tall tiles, of all of them and half the channels, so that weights are read once and not by
// two row tiles that soon drift apart.  Without / with them in us, 128 experts of 264 rows: 4096 x 7168 1676 / 1517, 4096 x
// 1024 286 / 273; of 384 and 448 rows 4096 x 7168: 1575 / 1748, 1636 / 1943.  Without silu, where a tile has twice the
// results, they gain with a large inner size only (4096 x 4096 965 / 860, 7168 x 2048 719 / 759), and their being there costs
// every other shape 1 to 2 %.
constexpr int kTallBlocks = 5;
constexpr int kBigThreads = 256;
constexpr int kRowGroup = 8;
// A stage of the ring is 128 bytes of k: of the channels (32 KiB), then of the rows (8 KiB for 64 of them).  Tiles of few
// rows wait for memory and have room for a third stage.
constexpr int kRingBytes = 144 * 1024;
__host__ __device__ constexpr int channels_of(int blocks) { return blocks <= kMaxBlocks ? kBigN : kBigN / 2; }
__host__ __device__ constexpr int stage_bytes_of(int blocks) { return (channels_of(blocks) + blocks * kBlockRows) * kStageK; }
__host__ __device__ constexpr int stages_of(int blocks) { return blocks <= 2 ? 3 : 2; }
constexpr bool ring_holds(int blocks) { return stages_of(blocks) * stage_bytes_of(blocks) <= kRingBytes; }
static_assert(ring_holds(1) && ring_holds(2) && ring_holds(3) && ring_holds(4) && ring_holds(5),
              "the ring");
// Results of up to this many bytes are written through into the 256 MB memory-side cache where the weights pass that cache
// by (256 x 64 rows x 4096, 134 MB, k 4096: 698 us, streamed 737); more would push one another out (256 x 128 rows x 7168,
// 470 MB, k 2048: 840, streamed 768), and so do weights that go through it (8192^3: 471, streamed 442).
constexpr long long kCachedOutput = 192LL << 20;
constexpr int kTableAt = kRingBytes;    // row tiles before every thread's experts
constexpr int kRowScaleBytes = 2 * kBigThreads * 4;
static_assert(kTallBlocks * kBlockRows * 4 <= kRowScaleBytes, "a tile's row scales");
constexpr int kScaleBytes = kRowScaleBytes + kBigN * 4;
constexpr int kScalesAt = kTableAt + (kBigThreads + 4) * 4;  // two tiles' row and channel scales
constexpr int kBigLds = kScalesAt + 2 * kScaleBytes;
static_assert(kBigLds <= 160 * 1024, "one workgroup takes a compute unit's LDS");

// Row tiles of a segment of so many pairs of blocks: as few as possible, each with blocks / tiles of them, rounded
// down or up.
__device__ __forceinline__ int row_tiles_of(int blocks) { return (blocks + kMaxBlocks - 1) / kMaxBlocks; }

struct BigTile {
  int expert, column;  // first output column
  int first, rows;     // rows of a
  int only;            // no other tile has rows of the expert
};

// One workgroup's walk over its tiles.  Wave (mw, nw) owns the 32-row blocks mw, mw + 2, ... and half, 128, of the 256
// channels (with kSilu 64 gate channels and the 64 up channels of the same columns; of a tall tile half as many).
template <bool kSilu>
struct BigMatmul {
  static constexpr int kColumns = kSilu ? kBigN / 2 : kBigN;  // output columns of a tile
  const ExpertMatmulArgs& a;
  unsigned char* const lds;
  const int lds_base, lane, wave, mw, nw, K, columns, steps;
  const bool stream_output;
  int4v desc_a, desc_b;

  // The same value, but not the same for the compiler: what is derived from it is computed where it is used
  // instead of being kept in registers across the tile loop, where it would be spilled.
  static __device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
  }
  __device__ __forceinline__ BigMatmul(const ExpertMatmulArgs& args, unsigned char* shared)
      : a(args),
        lds(shared),
        lds_base(lds_address(shared)),
        lane(lane_id()),
        wave(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6)),
        mw(wave & 1),
        nw(wave >> 1),
        K(args.in_features),
        columns(kSilu ? args.out_features / 2 : args.out_features),
        steps((args.in_features + kStageK - 1) / kStageK),
        stream_output(static_cast<long long>(args.num_rows) * columns > kCachedOutput / 2) {}

  // Channels of a tile as 32-wide blocks of a wave, of a matrix, and as output columns.
  template <int kBlocks>
  static constexpr int kChannels = channels_of(kBlocks) / 64;
  template <int kBlocks>
  static constexpr int kOut = channels_of(kBlocks) / (kSilu ? 2 : 1);

  // Load j of stage `step`, whose place in the ring is `slot`: eight rows of the channels, or of the tokens.
  template <bool kOnce, int kPerWave>
  __device__ __forceinline__ void load_b(const Place& at, int slot, int step, int j) const {
    const int row = (kSilu ? wave & 1 : wave) * (8 * kPerWave) + at.row + j * 8, piece = at.piece_of(j);
    load_to_lds<kOnce>(desc_b, lds_base + slot + (wave * kPerWave + j) * kChunkBytes,
                       step * kStageK + piece < K ? row * K + piece : kOutside, step * kStageK);
  }
  __device__ __forceinline__ void load_a(const Place& at, int slot, int step, int j) const {
    const int eight = (j >> 1) * 8 + wave * 2 + (j & 1), piece = at.piece_of(j);
    load_to_lds(desc_a, lds_base + slot + eight * kChunkBytes,
                step * kStageK + piece < K ? (eight * 8 + at.row) * K + piece : kOutside, step * kStageK);
  }

  // Points the descriptors at a tile and starts the loads of its scales and of its first stages, as many as the ring holds.
  __device__ __forceinline__ void start(const BigTile& tile, int scales_at) {
    const int blocks = (tile.rows + kBlockRows - 1) / kBlockRows;
    const bool tall = kSilu && blocks > kMaxBlocks;
    const int channels = tall ? kBigN / 2 : kBigN, width = tall ? kColumns / 2 : kColumns, left = columns - tile.column;
    const int b_rows = left >= width ? width : tall && left < 0 ? 0 : left;
    const size_t channel = static_cast<size_t>(tile.expert) * a.out_features + (kSilu && wave >= 2 ? columns : 0) + tile.column;
    desc_a = descriptor_of(a.a + static_cast<size_t>(tile.first) * K, tile.rows * K);
    desc_b = descriptor_of(a.b + channel * K, b_rows * K);
    const int stride = static_cast<int>(a.a_scales_row_stride);
    const Place at(fresh(lane));
    const int row = fresh(static_cast<int>(threadIdx.x));
    const int4v desc_scales = descriptor_of(a.a_scales + static_cast<size_t>(tile.first) * a.a_scales_row_stride,
                                            ((tile.rows - 1) * stride + 1) * 4);
    load_word_to_lds(desc_scales, scales_at + wave * 256, row < tile.rows ? row * stride * 4 : kOutside);
    if constexpr (kSilu)
      load_word_to_lds(desc_scales, scales_at + (kBigThreads + wave * 64) * 4,
                       row + kBigThreads < tile.rows ? (row + kBigThreads) * stride * 4 : kOutside);
    load_word_to_lds(descriptor_of(a.b_scales + channel, b_rows * 4), scales_at + kRowScaleBytes + wave * 256,
                     (kSilu ? row & 127 : row) * 4);
    const int stages = stages_of(blocks), stage_bytes = (channels + blocks * kBlockRows) * kStageK;
    for (int s = 0; s < stages && s < steps; ++s) {
      const int slot = s * stage_bytes;
      if (tall) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load_b<true, 4>(at, slot, s, j);
      } else if (tile.only != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) load_b<true, 8>(at, slot, s, j);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) load_b<false, 8>(at, slot, s, j);
      }
#pragma unroll
      for (int j = 0; j < 2 * (kSilu ? kTallBlocks : kMaxBlocks); ++j)
        if (j < 2 * blocks) load_a(at, slot + channels * kStageK, s, j);
    }
  }

  template <int kBlocks>
  struct Fragments {
    int4v a[2][kBlocks], b[2][kChannels<kBlocks>];
  };
  // Fragment i of a quarter of a stage: the wave's channels, then the rows.  Lane l takes row l % 32 of a block and
  // piece 2 * quarter + l / 32.
  template <int kBlocks>
  __device__ __forceinline__ void read(const Place& at, Fragments<kBlocks>& f, int slot, int quarter, int i) const {
    constexpr int kCh = kChannels<kBlocks>;
    const unsigned char* base = lds + slot + (at.read_at ^ (quarter * 32));
    if (i < kCh) {
      const int block = kSilu ? i % (kCh / 2) + nw * (kCh / 2) + i / (kCh / 2) * kCh : nw * kCh + i;
      f.b[quarter & 1][i] = *reinterpret_cast<const int4v*>(base + block * 32 * kStageK);
    } else {
      f.a[quarter & 1][i - kCh] =
          *reinterpret_cast<const int4v*>(base + (channels_of(kBlocks) + (2 * (i - kCh) + mw) * 32) * kStageK);
    }
  }

  enum Loads { kNone, kWeights, kRows };
  // A quarter of a stage's products; between them, spread over them, the reads of the next quarter's fragments (from
  // the stage in `from`, or with kRead false none) and the loads of a part of stage `ahead` (to `to`).
  template <int kBlocks, bool kOnce, int kQuarter, Loads kLoad, bool kRead = true>
  __device__ __forceinline__ void quarter(const Place& at, Fragments<kBlocks>& f, int16v (&acc)[kBlocks][kChannels<kBlocks>], int from, int to,
                                          int ahead) const {
    constexpr int kCh = kChannels<kBlocks>;
    constexpr int kLoads = kLoad == kNone ? 0 : kLoad == kWeights ? 2 * kCh : 2 * kBlocks;
    constexpr int kProducts = kCh * kBlocks, kItems = (kRead ? kCh + kBlocks : 0) + kLoads;
#pragma unroll
    for (int p = 0; p < kProducts; ++p) {
#pragma unroll
      for (int i = p * kItems / kProducts; i < (p + 1) * kItems / kProducts; ++i) {
        const int loads_before = kLoads == 0 ? 0 : (i + 1) * kLoads / kItems;
        const bool is_load = kLoads != 0 && loads_before != i * kLoads / kItems;
        if (is_load) kLoad == kWeights ? load_b<kOnce, 2 * kCh>(at, to, ahead, loads_before - 1)
                                   : load_a(at, to + channels_of(kBlocks) * kStageK, ahead, loads_before - 1);
        else read<kBlocks>(at, f, from, (kQuarter + 1) & 3, i - loads_before);
      }
      constexpr int h = kQuarter & 1;
      acc[p / kCh][p % kCh] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.b[h][p % kCh], f.a[h][p / kCh], acc[p / kCh][p % kCh], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The products of one tile whose rows fill kBlocks pairs of 32-row blocks, the start of the next tile, and
  // the epilogue.
  template <int kBlocks, bool kOnce>
  __device__ __forceinline__ void run(const BigTile& tile, int scales_at, bool has_next, const BigTile& next, int next_scales_at) {
    const Place at(fresh(lane));
    constexpr int kCh = kChannels<kBlocks>;
    int16v acc[kBlocks][kCh];
    Fragments<kBlocks> f;
#pragma unroll
    for (int m = 0; m < kBlocks; ++m)
#pragma unroll
      for (int j = 0; j < kCh; ++j) acc[m][j] = int16v{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

    constexpr int kStages = stages_of(kBlocks), kStageBytes = stage_bytes_of(kBlocks), kStageLoads = 2 * kCh + 2 * kBlocks;
    if (steps >= kStages)
      wait_and_meet<(kStages - 1) * kStageLoads + kStores>();
    else
      wait_and_meet<kStores>();
#pragma unroll
    for (int i = 0; i < kCh + kBlocks; ++i) read<kBlocks>(at, f, 0, 0, i);
    quarter<kBlocks, kOnce, 0, kNone>(at, f, acc, 0, 0, 0);
    quarter<kBlocks, kOnce, 1, kNone>(at, f, acc, 0, 0, 0);
    quarter<kBlocks, kOnce, 2, kNone>(at, f, acc, 0, 0, 0);
    // The barrier behind the third quarter of stage s makes stage s + 1 visible (younger ones and at first the previous
    // tile's stores may still be on their way), and tells that every wave has read all of stage s, whose place stage
    // s + kStages then fills.
    int step = 0, here = 0;
    const auto after = [](int slot) { return slot == (kStages - 1) * kStageBytes ? 0 : slot + kStageBytes; };
    const auto go_on = [&](auto load) {
      constexpr bool kLoad = decltype(load)::value;
      const int next_slot = after(here), ahead = step + kStages;
      quarter<kBlocks, kOnce, 3, kLoad ? kWeights : kNone>(at, f, acc, next_slot, here, ahead);
      quarter<kBlocks, kOnce, 0, kLoad ? kRows : kNone>(at, f, acc, next_slot, here, ahead);
      quarter<kBlocks, kOnce, 1, kNone>(at, f, acc, next_slot, 0, 0);
      quarter<kBlocks, kOnce, 2, kNone>(at, f, acc, next_slot, 0, 0);
      ++step;
      here = next_slot;
    };
    while (step < kStages - 1 && step + kStages < steps) {
      wait_and_meet<(kStages - 2) * kStageLoads + kStores>();
      go_on(std::true_type{});
    }
    while (step + kStages < steps) {
      wait_and_meet<(kStages - 2) * kStageLoads>();
      go_on(std::true_type{});
    }
    while (step + 1 < steps) {  // steps - step - 2 stages are behind the next one
      if (steps - step > 2) wait_and_meet<(kStages - 2) * kStageLoads>();
      else wait_and_meet<0>();
      go_on(std::false_type{});
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
    quarter<kBlocks, kOnce, 3, kNone, false>(at, f, acc, 0, 0, 0);
    // The next tile's loads run during this one's epilogue.
    if (has_next) start(next, next_scales_at);

    // Lane l holds row l % 32 of a block and channels 8 g + 4 (l / 32) + 0..3.
    const int lane = fresh(this->lane), r = lane & 31;
    const float* row_scales = reinterpret_cast<const float*>(lds + (scales_at - lds_base));
    const float* b_scales = row_scales + kRowScaleBytes / 4;
    const __amdgpu_buffer_rsrc_t out = out_rows(tile);
    const int store_row = lane & 15, store_column = ((lane >> 5) + ((lane >> 3) & 2)) * 8;
    float row_scale[kBlocks];
#pragma unroll
    for (int m = 0; m < kBlocks; ++m) row_scale[m] = row_scales[(2 * m + mw) * 32 + r];
#pragma unroll
    for (int j = 0; j < (kSilu ? kCh / 2 : kCh); ++j) {
      const int column0 = nw * (kOut<kBlocks> / 2) + j * 32;  // in the tile
      float4 s[4], u[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        s[g] = *reinterpret_cast<const float4*>(b_scales + column0 + g * 8 + (lane >> 5) * 4);
        if constexpr (kSilu) u[g] = *reinterpret_cast<const float4*>(b_scales + 128 + column0 + g * 8 + (lane >> 5) * 4);
      }
      const int column = tile.column + column0 + store_column;
#pragma unroll
      for (int m = 0; m < kBlocks; ++m) {
        uint32_t w[4][2];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float sg[4] = {s[g].x, s[g].y, s[g].z, s[g].w};
          float o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = static_cast<float>(acc[m][j][g * 4 + i]) * (row_scale[m] * sg[i]);
          if constexpr (kSilu) {
            const float ug[4] = {u[g].x, u[g].y, u[g].z, u[g].w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[i] = silu(o[i]) * (static_cast<float>(acc[m][(j + kCh / 2) % kCh][g * 4 + i]) * (row_scale[m] * ug[i]));
          }
          w[g][0] = to_bf16_pair(o[0], o[1]);
          w[g][1] = to_bf16_pair(o[2], o[3]);
        }
        // Exchanges between the halves of the wave give a lane eight columns in a row: l < 32 those of g = 0 (2), the others those
        // of g = 1 (3); between groups of 16 lanes, 16 rows of 64 bytes to a store.
        vec16 first, second;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto low = __builtin_amdgcn_permlane32_swap(w[0][i], w[1][i], false, false);
          const auto high = __builtin_amdgcn_permlane32_swap(w[2][i], w[3][i], false, false);
          const auto even = __builtin_amdgcn_permlane16_swap(low[0], high[0], false, false);
          const auto odd = __builtin_amdgcn_permlane16_swap(low[1], high[1], false, false);
          first[i] = even[0], first[2 + i] = odd[0], second[i] = even[1], second[2 + i] = odd[1];
        }
        const int row = (2 * m + mw) * 32 + store_row;
        const bool inside = column < columns;
        const int at_first = inside ? (row * columns + column) * 2 : kOutside;
        const int at_second = inside ? ((row + 16) * columns + column) * 2 : kOutside;
        if (!kOnce || stream_output) {
          __builtin_amdgcn_raw_buffer_store_b128(first, out, at_first, 0, kCachePolicyDeviceScope | kCachePolicyStreaming);
          __builtin_amdgcn_raw_buffer_store_b128(second, out, at_second, 0, kCachePolicyDeviceScope | kCachePolicyStreaming);
        } else {
          __builtin_amdgcn_raw_buffer_store_b128(first, out, at_first, 0, kCachePolicyDeviceScope);
          __builtin_amdgcn_raw_buffer_store_b128(second, out, at_second, 0, kCachePolicyDeviceScope);
        }
        __builtin_amdgcn_sched_barrier(0);  // one block's values at a time: more would not fit the registers
      }
    }
    idle_stores<kStores - 2 * kBlocks * (kSilu ? kCh / 2 : kCh)>(out);
  }

  // The waits of the next tile's first steps count the stores of this one, so every tile issues as many: rows
  // behind the tile's and columns behind the matrix lie outside the descriptor and go nowhere.
  static constexpr int kStores = kMaxBlocks * (kSilu ? 4 : 8);
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t out_rows(const BigTile& tile) const {
    return __builtin_amdgcn_make_buffer_rsrc(a.out + static_cast<size_t>(tile.first) * columns, 0, tile.rows * columns * 2,
                                             kRawBufferFormat);
  }
  template <int kCount>
  __device__ __forceinline__ void idle_stores(__amdgpu_buffer_rsrc_t out) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) __builtin_amdgcn_raw_buffer_store_b128(vec16{0, 0, 0, 0}, out, kOutside, i, 0);
  }
  // Until at most kYounger of the wave's memory operations are on their way and its LDS reads are back, then
  // until every wave got there.
  template <int kYounger>
  static __device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(kYounger) : "memory");
  }
};

template <bool kSilu>
__global__ __launch_bounds__(kBigThreads, 1) void ep_expert_matmul_big_kernel(const ExpertMatmulArgs a) {
  extern __shared__ __align__(1024) unsigned char lds[];
  constexpr int kPer = kMaxExperts / kBigThreads;
  int* tiles_before = reinterpret_cast<int*>(lds + kTableAt);  // [kBigThreads + 1], before the experts of every thread
  const int t = static_cast<int>(threadIdx.x);
  const int per = (a.num_experts + kBigThreads - 1) / kBigThreads;
  const auto tiles_of = [&](int e) {
    return e < a.num_experts ? row_tiles_of((segment_of(a, e).rows + kBlockRows - 1) / kBlockRows) : 0;
  };
  {
    int* wave_total = reinterpret_cast<int*>(lds);
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) mine += j < per ? tiles_of(t * per + j) : 0;
    const int upto = wave_inclusive_scan(mine);
    if (lane_id() == kWave - 1) wave_total[t >> 6] = upto;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < (t >> 6); ++w) before += wave_total[w];
    tiles_before[t] = before;
    if (t == kBigThreads - 1) tiles_before[kBigThreads] = before + mine;
    __syncthreads();
  }
  BigMatmul<kSilu> matmul(a, lds);
  constexpr int kColumns = BigMatmul<kSilu>::kColumns;
  const int column_tiles = (matmul.columns + kColumns - 1) / kColumns;
  const auto locate = [&](int index) {
    const int row_tile_times = index / column_tiles;
    int lo = 0, hi = kBigThreads;  // tiles_before[lo] <= row_tile_times < tiles_before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (__builtin_amdgcn_readfirstlane(tiles_before[mid]) <= row_tile_times) lo = mid;
      else hi = mid;
    }
    int first_tile = __builtin_amdgcn_readfirstlane(tiles_before[lo]);
    int expert = lo * per;
    for (int j = 1; j < per; ++j) {  // up to three more experts of the same thread
      const int tiles = __builtin_amdgcn_readfirstlane(tiles_of(expert));
      if (first_tile + tiles > row_tile_times) break;
      first_tile += tiles;
      ++expert;
    }
    const Segment all = segment_of(a, expert);
    const int rows = __builtin_amdgcn_readfirstlane(all.rows);
    const int blocks = (rows + kBlockRows - 1) / kBlockRows, row_tiles = row_tiles_of(blocks);
    if (kSilu && blocks == kTallBlocks)  // in the place of two row tiles
      return BigTile{expert, (index - first_tile * column_tiles) * (kColumns / 2), __builtin_amdgcn_readfirstlane(all.first), rows, 1};
    // Inside an expert: groups of up to eight row tiles by as many columns as make about 32 tiles, one die's share
    // at a time, so that rows and weights are each fetched once for all of them; columns fastest, so that a
    // group's shorter tiles are shared out over all compute units and not always to the same ones.
    const int inside = index - first_tile * column_tiles;
    const int group = inside / (kRowGroup * column_tiles);
    const int in_group = inside - group * kRowGroup * column_tiles;
    const int rows_left = row_tiles - group * kRowGroup;
    const int group_rows = rows_left < kRowGroup ? rows_left : kRowGroup;
    const int chunk_columns = 32 / group_rows;
    const int chunk = in_group / (group_rows * chunk_columns);
    const int in_chunk = in_group - chunk * group_rows * chunk_columns;
    const int columns_left = column_tiles - chunk * chunk_columns;
    const int width = columns_left < chunk_columns ? columns_left : chunk_columns;
    const int row_in_group = in_chunk / width;
    const int row_tile = group * kRowGroup + row_in_group, column_tile = chunk * chunk_columns + in_chunk - row_in_group * width;
    const int from = static_cast<int>(static_cast<long long>(row_tile) * blocks / row_tiles) * kBlockRows;
    const int to = static_cast<int>(static_cast<long long>(row_tile + 1) * blocks / row_tiles) * kBlockRows;
    return BigTile{expert, column_tile * kColumns, __builtin_amdgcn_readfirstlane(all.first) + from,
                   (to < rows ? to : rows) - from, row_tiles == 1 ? 1 : 0};
  };

  // Workgroups go to the eight dies in turn; each die takes one contiguous run of the tiles, so that the rows
  // and weights its compute units share come from its own L2.
  // Segments that do not overlap make no more tiles than this; what overlapping ones (tables of a layout that gave
  // up) would make beyond is not computed.
  const int most = a.num_rows / (kMaxBlocks * kBlockRows) + a.num_experts;
  const int made = __builtin_amdgcn_readfirstlane(tiles_before[kBigThreads]);
  const int total = (made < most ? made : most) * column_tiles;
  const int dies = gridDim.x % 8 == 0 ? 8 : 1;
  const int per_die = (total + dies - 1) / dies;
  const int die = static_cast<int>(blockIdx.x) % dies;
  const int end = (die + 1) * per_die < total ? (die + 1) * per_die : total;
  const int stride = static_cast<int>(gridDim.x) / dies;
  int index = die * per_die + static_cast<int>(blockIdx.x) / dies;
  if (index >= end) return;
  const int scales_at = matmul.lds_base + kScalesAt;
  int turn = 0;
  BigTile tile = locate(index);
  matmul.start(tile, scales_at);
  matmul.template idle_stores<BigMatmul<kSilu>::kStores>(matmul.out_rows(tile));
  for (;;) {
    index += stride;
    const bool has_next = index < end;
    const BigTile next = has_next ? locate(index) : tile;
    const int at = scales_at + turn * kScaleBytes, next_at = scales_at + (turn ^ 1) * kScaleBytes;
    const int blocks = (tile.rows + kBlockRows - 1) / kBlockRows;
    if (tile.only != 0) switch (blocks) {
      case 1: matmul.template run<1, true>(tile, at, has_next, next, next_at); break;
      case 2: matmul.template run<2, true>(tile, at, has_next, next, next_at); break;
      case 3: matmul.template run<3, true>(tile, at, has_next, next, next_at); break;
      case 4: matmul.template run<4, true>(tile, at, has_next, next, next_at); break;
      default:
        if constexpr (kSilu) matmul.template run<5, true>(tile, at, has_next, next, next_at);
        break;
    }
    else switch (blocks) {  // the shares of at least five blocks
      case 2: matmul.template run<2, false>(tile, at, has_next, next, next_at); break;
      case 3: matmul.template run<3, false>(tile, at, has_next, next, next_at); break;
      default: matmul.template run<4, false>(tile, at, has_next, next, next_at); break;
    }
    if (!has_next) return;
    tile = next;
    turn ^= 1;
  }
}

}  // namespace

hipError_t launch_expert_matmul(const ExpertMatmulArgs& a, hipStream_t stream) {
  if (a.num_rows == 0) return hipSuccess;
  const int columns = a.silu_mul ? a.out_features / 2 : a.out_features;
  // Large tiles where there are enough of them for most compute units and enough rows in each to be worth the
  // accumulators.  Small / large in us: 256 experts x 4096 x 7168 with 4, 8, 16, 32 rows each: 1127 / 1128, 1145 / 1135,
  // 1128 / 1099, 1232 / 1181; 64 large tiles (8 x 256 rows x 2048 channels, k 2048): 31 / 31, (1024 rows x 4096, k 4096):
  // 36 / 44; 96 (8 x 384 x 2048, k 2048): 44 / 31; 128 (8 x 256 x 4096, k 2048): 57 / 35.
  const long long big_columns = a.silu_mul ? kBigN / 2 : kBigN;
  const long long by_rows = a.num_rows / (kMaxBlocks * kBlockRows);
  const long long by_experts = a.num_rows / 12 < a.num_experts ? a.num_rows / 12 : a.num_experts;
  const long long big_tiles = (by_rows > by_experts ? by_rows : by_experts) * ((columns + big_columns - 1) / big_columns);
  const bool big = a.num_rows > 12LL * a.num_experts && big_tiles >= 96;
  if (big) {
    DeviceTraits dev{};
    hipError_t err = device_traits(stream, &dev);
    if (err != hipSuccess) return err;
    static LdsCeiling ceilings[2];
    const void* kernel = a.silu_mul ? reinterpret_cast<const void*>(&ep_expert_matmul_big_kernel<true>)
                                    : reinterpret_cast<const void*>(&ep_expert_matmul_big_kernel<false>);
    err = ceilings[a.silu_mul ? 1 : 0].raise(kernel, kBigLds, stream);
    if (err != hipSuccess) return err;
    const dim3 grid(static_cast<unsigned>(dev.compute_units));
    if (a.silu_mul)
      hipLaunchKernelGGL((ep_expert_matmul_big_kernel<true>), grid, dim3(kBigThreads), kBigLds, stream, a);
    else
      hipLaunchKernelGGL((ep_expert_matmul_big_kernel<false>), grid, dim3(kBigThreads), kBigLds, stream, a);
    return hipGetLastError();
  }
  // Every segment ends in at most one partial tile.
  const int row_tiles = a.num_rows / kTileM + a.num_experts;
  const unsigned column_tiles = static_cast<unsigned>((columns + kTileN - 1) / kTileN);
  if (a.silu_mul)
    hipLaunchKernelGGL((ep_expert_matmul_small_kernel<true>), dim3(column_tiles, static_cast<unsigned>(row_tiles)),
                       dim3(kSmallThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((ep_expert_matmul_small_kernel<false>), dim3(column_tiles, static_cast<unsigned>(row_tiles)),
                       dim3(kSmallThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mi_ep
