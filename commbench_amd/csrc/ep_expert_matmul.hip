// The experts' products on dispatched rows, int8 x int8 with a scale for each row and each output
// channel, for gfx950:
//   c[m, n] = a_scale[m] * b_scale[e, n] * sum_k a[m, k] * b[e, n, k]     rows m of expert e's segment
//   out = bf16(c)   or, gate and up in one product,   out[m, i] = bf16(silu(c[m, i]) * c[m, I + i])
// The sum over k is exact in 32-bit integers (|a|, |b| <= 128 and k < 2^17).
#include "ep_device.h"

namespace mi_ep {
namespace {

typedef int int4v __attribute__((ext_vector_type(4)));

constexpr int kTileM = 64, kTileN = 64, kStepK = 64;
constexpr int kPitch = kStepK + 16;  // bytes between LDS rows: 16-byte reads of 16 rows meet different banks

struct RowTile {
  int expert, first, rows;  // rows [first, first + rows) of a and out; rows == 0: no such tile
};

// The `index`-th tile of up to kTileM rows, the experts' segments cut into tiles one after the other.
// Segments are clamped to [0, num_rows), whatever the tables hold.
__device__ __forceinline__ RowTile find_row_tile(const ExpertMatmulArgs& a, int index) {
  __shared__ int wave_tiles[4];
  __shared__ RowTile found;
  const int t = static_cast<int>(threadIdx.x);
  const int per = (a.num_experts + 255) / 256;
  if (t == 0) found = RowTile{0, 0, 0};
  int mine = 0;
  const auto segment = [&](int e, int* first) {
    long long lo = 0, hi = a.num_rows;
    if (a.expert_offsets != nullptr) {
      lo = a.expert_offsets[e];
      hi = a.num_tokens_per_expert != nullptr ? lo + a.num_tokens_per_expert[e] : a.expert_offsets[e + 1];
    }
    if (lo < 0) lo = 0;
    if (hi > a.num_rows) hi = a.num_rows;
    *first = static_cast<int>(lo);
    return hi > lo ? static_cast<int>(hi - lo) : 0;
  };
  for (int j = 0; j < per; ++j) {
    const int e = t * per + j;
    int first;
    if (e < a.num_experts) mine += (segment(e, &first) + kTileM - 1) / kTileM;
  }
  const int upto = wave_inclusive_scan(mine);
  if (lane_id() == kWave - 1) wave_tiles[t >> 6] = upto;
  __syncthreads();
  int before = upto - mine;
  for (int w = 0; w < (t >> 6); ++w) before += wave_tiles[w];
  if (index >= before && index < before + mine) {
    for (int j = 0; j < per; ++j) {
      const int e = t * per + j;
      int first = 0;
      const int rows = e < a.num_experts ? segment(e, &first) : 0;
      const int tiles = (rows + kTileM - 1) / kTileM;
      if (index >= before && index < before + tiles) {
        const int skip = (index - before) * kTileM;
        found = RowTile{e, first + skip, rows - skip < kTileM ? rows - skip : kTileM};
      }
      before += tiles;
    }
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }

// One workgroup: 64 rows by 64 output columns (with kSilu the 64 gate and the 64 up channels of those
// columns).  Wave w owns 16 output columns.
template <bool kSilu>
__global__ __launch_bounds__(256) void ep_expert_matmul_kernel(const ExpertMatmulArgs a) {
  constexpr int kSets = kSilu ? 2 : 1;
  __shared__ __align__(16) unsigned char stage_a[kTileM * kPitch];
  __shared__ __align__(16) unsigned char stage_b[kSets * kTileN * kPitch];
  const RowTile tile = find_row_tile(a, static_cast<int>(blockIdx.y));
  if (tile.rows == 0) return;
  const int out_columns = kSilu ? a.out_features / 2 : a.out_features;
  const int n0 = static_cast<int>(blockIdx.x) * kTileN;
  const int t = static_cast<int>(threadIdx.x), lane = lane_id(), wave = t >> 6;
  const int load_row = t >> 2, load_k = (t & 3) * 16;

  const unsigned char* a_row = a.a + static_cast<size_t>(tile.first + (load_row < tile.rows ? load_row : 0)) * a.in_features;
  const int n_row = n0 + load_row < out_columns ? n0 + load_row : out_columns - 1;
  const unsigned char* b_row =
      a.b + (static_cast<size_t>(tile.expert) * a.out_features + n_row) * a.in_features;

  int4v acc[kSets][kTileM / 16];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int m = 0; m < kTileM / 16; ++m) acc[s][m] = int4v{0, 0, 0, 0};

  for (int k0 = 0; k0 < a.in_features; k0 += kStepK) {
    const bool inside = k0 + load_k < a.in_features;
    const vec16 zero = {0, 0, 0, 0};
    *reinterpret_cast<vec16*>(stage_a + load_row * kPitch + load_k) =
        inside ? *reinterpret_cast<const vec16*>(a_row + k0 + load_k) : zero;
#pragma unroll
    for (int s = 0; s < kSets; ++s)
      *reinterpret_cast<vec16*>(stage_b + (s * kTileN + load_row) * kPitch + load_k) =
          inside ? *reinterpret_cast<const vec16*>(b_row + static_cast<size_t>(s) * out_columns * a.in_features + k0 + load_k)
                 : zero;
    __syncthreads();
    int4v w[kSets];
#pragma unroll
    for (int s = 0; s < kSets; ++s)
      w[s] = *reinterpret_cast<const int4v*>(stage_b + (s * kTileN + wave * 16 + (lane & 15)) * kPitch + (lane >> 4) * 16);
#pragma unroll
    for (int m = 0; m < kTileM / 16; ++m) {
      const int4v x = *reinterpret_cast<const int4v*>(stage_a + (m * 16 + (lane & 15)) * kPitch + (lane >> 4) * 16);
#pragma unroll
      for (int s = 0; s < kSets; ++s) acc[s][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[s], x, acc[s][m], 0, 0, 0);
    }
    __syncthreads();
  }

  // Lane l holds channels 4 * (l / 16) .. + 3 of row l % 16 of every 16 x 16 product.
  const int n = n0 + wave * 16 + (lane >> 4) * 4;
  if (n >= out_columns) return;
  const float* b_scales = a.b_scales + static_cast<size_t>(tile.expert) * a.out_features + n;
#pragma unroll
  for (int m = 0; m < kTileM / 16; ++m) {
    const int r = m * 16 + (lane & 15);
    if (r >= tile.rows) continue;
    const float row_scale = a.a_scales[static_cast<size_t>(tile.first + r) * a.a_scales_row_stride];
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = static_cast<float>(acc[0][m][i]) * (row_scale * b_scales[i]);
      if constexpr (kSilu) o[i] = silu(o[i]) * (static_cast<float>(acc[kSets - 1][m][i]) * (row_scale * b_scales[out_columns + i]));
    }
    *reinterpret_cast<uint2*>(a.out + static_cast<size_t>(tile.first + r) * out_columns + n) =
        uint2{pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
  }
}

}  // namespace

hipError_t launch_expert_matmul(const ExpertMatmulArgs& a, hipStream_t stream) {
  if (a.num_rows == 0) return hipSuccess;
  const int columns = a.silu_mul ? a.out_features / 2 : a.out_features;
  // Every segment ends in at most one partial tile.
  const int row_tiles = a.num_rows / kTileM + a.num_experts;
  if (row_tiles > 65535) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>((columns + kTileN - 1) / kTileN), static_cast<unsigned>(row_tiles));
  if (a.silu_mul)
    hipLaunchKernelGGL((ep_expert_matmul_kernel<true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((ep_expert_matmul_kernel<false>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mi_ep
