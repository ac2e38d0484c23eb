// Rows to 8 bits and back, for gfx950: the norm that makes an 8-bit dispatch payload, the
// requantisation between an expert's two products, and reading 8-bit rows back.
//
//   h = x + residual;  y = h / sqrt(mean(h^2) + eps) * weight      (or y = x: plain quantisation)
//   s = max|y| / qmax over the row (int8, qmax 127) or over 128 columns (e4m3, qmax 448); 1 if that is 0
//   q = round(y / s), ties to even
//
// A row is read once and stays in registers: one workgroup (rows up to 4096 columns: one wave) owns a
// row, so the mean and the maximum are two reductions over data that never leave the compute unit.  The
// sum of squares, the mean and y are fp32; nothing is rounded to bf16 on the way to q.  A row whose sum of squares leaves
// fp32 at either end is brought near one by a power of two, from the registers, and summed again.  Bound by HBM: 7
// bytes an element move (x, residual in, residual out, q) for about 25 vector instructions per 8 elements
// and reduction step.
#include "ep_expert.h"

namespace mi_ep {
namespace {

constexpr int kQuantBlockLanes = kQuantBlock / 8;  // lanes whose vectors share an e4m3 scale
static_assert(kQuantBlockLanes == 16, "the block maximum is a reduction over one row of 16 lanes");

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Sum / maximum over the 64 lanes by data-parallel-primitive moves (zero stands in for lanes without a
// source, which changes neither a sum nor a maximum of unsigned values); every lane gets the result.
__device__ __forceinline__ float wave_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x111, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x112, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x114, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x118, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x142, 0xa, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x143, 0xc, 0xf, false));
  return wave_read(v, kWave - 1);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x111, 0xf, 0xf, false)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x112, 0xf, 0xf, false)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x114, 0xf, 0xf, false)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x118, 0xf, 0xf, false)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x142, 0xa, 0xf, false)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x143, 0xc, 0xf, false)));
  return static_cast<uint32_t>(wave_read(static_cast<int>(v), kWave - 1));
}
// Maximum over each row of 16 lanes, in all of them (rotations inside the row).
__device__ __forceinline__ uint32_t block_max(uint32_t v) {
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x128, 0xf, 0xf, true)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x124, 0xf, 0xf, true)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x122, 0xf, 0xf, true)));
  v = umax(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x121, 0xf, 0xf, true)));
  return v;
}

// The same over a row's waves, through one word of LDS each.  A second call on the same words needs a barrier between
// the first's reads and its own writes.
template <int kWaves>
__device__ __forceinline__ float row_sum(float v, float* words, int wave) {
  v = wave_sum(v);
  if constexpr (kWaves > 1) {
    if (lane_id() == 0) words[wave] = v;
    __syncthreads();
    v = words[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += words[w];
  }
  return v;
}
template <int kWaves>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* words, int wave) {
  v = wave_max(v);
  if constexpr (kWaves > 1) {
    if (lane_id() == 0) words[wave] = v;
    __syncthreads();
    v = words[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = umax(v, words[w]);
  }
  return v;
}

// y / scale, correctly rounded: with r the rounded reciprocal of the scale, y * r corrected once by its
// own remainder (Markstein) is the rounded quotient as long as nothing leaves the normal range, which
// scales from 2^-100 on guarantee for every quotient that matters (larger than 2^-20).  Three instructions where
// the division takes ten; scales out of that range divide.
struct Divisor {
  float scale, reciprocal;
  __device__ __forceinline__ explicit Divisor(float s) : scale(s), reciprocal(1.0f / s) {}
  __device__ __forceinline__ bool in_range() const { return scale >= 0x1p-100f && scale <= 0x1p100f; }
  __device__ __forceinline__ float operator()(float y) const {
    const float q = y * reciprocal;
    return __builtin_fmaf(__builtin_fmaf(-q, scale, y), reciprocal, q);
  }
};

// Codes on their way to the expert's next product: written through into the memory-side cache (65536 x 2048 and read back:
// 133.9 us left to the L2s, 131.3; 16384 x 2048 e4m3: 37.9 and 36.3).  The norm's, which are a small part of what it
// writes, are left to the L2s (4096 x 4096: 32.3 us, written through 33.2).
template <bool kNorm>
__device__ __forceinline__ void store_codes(uint2* to, uint2 codes) {
  if constexpr (kNorm)
    *to = codes;
  else
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), static_cast<uint64_t>(codes.y) << 32 | codes.x, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}

template <int kFormat>
constexpr float kLargestCode = kFormat == kQuantInt8 ? 127.0f : 448.0f;
// The scale of values whose largest magnitude has these bits.  Infinities and NaN order above every
// finite value as integers, so a row (block) that holds one gets a NaN scale and reads back as NaN
// throughout instead of as something finite.  A scale of zero, of values so small that the quotient vanishes too, is 1.
template <int kFormat>
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits >= 0x7f800000u ? 0x7fc00000u : amax_bits);
  const float scale = amax / kLargestCode<kFormat>;
  return scale == 0.0f ? 1.0f : scale;
}

template <int kFormat>
__device__ __forceinline__ uint2 codes8(const float (&q)[8]) {
  uint2 out;
  if constexpr (kFormat == kQuantInt8) {
    // Added to 1.5 * 2^23 a quotient is rounded to a whole number, ties to even, whose two's complement is in the
    // low byte; NaN gives some code, which its NaN scale makes NaN again.
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(q[i] + 12582912.0f);
    out.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u),
                                  0x05040100u);
    out.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[7], b[6], 0x0c0c0400u), __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400u),
                                  0x05040100u);
  } else {
    int lo = 0, hi = 0;  // the conversion rounds to nearest even; quotients end at 448
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    out.x = static_cast<uint32_t>(lo);
    out.y = static_cast<uint32_t>(hi);
  }
  return out;
}

template <int kFormat>
__device__ __forceinline__ uint2 quantize8(const float (&y)[8], const Divisor& divide) {
  float q[8];
  if (__builtin_expect(divide.in_range(), 1)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = divide(y[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // A subnormal scale has few digits: its quotients may lie beyond the largest code (NaN passes the comparisons).
      q[i] = y[i] / divide.scale;
      if (q[i] > kLargestCode<kFormat>) q[i] = kLargestCode<kFormat>;
      if (q[i] < -kLargestCode<kFormat>) q[i] = -kLargestCode<kFormat>;
    }
  }
  return codes8<kFormat>(q);
}

__device__ __forceinline__ void unpack8(const vec16 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16_lo(v[i]);
    f[2 * i + 1] = bf16_hi(v[i]);
  }
}
__device__ __forceinline__ vec16 pack8(const float (&f)[8]) {
  vec16 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_bf16_pair(f[2 * i], f[2 * i + 1]);
  return v;
}

// kRowThreads threads own a row of up to kRowThreads * kVecs vectors of 8 columns.
template <int kRowThreads, int kVecs, bool kNorm, int kFormat>
__global__ __launch_bounds__(kRowThreads == kWave ? 4 * kWave : kRowThreads) void ep_quantize_rows_kernel(
    const QuantizeArgs a) {
  constexpr int kRows = kRowThreads == kWave ? 4 : 1;
  constexpr int kWaves = kRowThreads / kWave;
  __shared__ float sums[kWaves];
  __shared__ uint32_t maxima[kWaves];
  const int t = kRows == 1 ? static_cast<int>(threadIdx.x) : lane_id();
  const int wave = static_cast<int>(threadIdx.x) >> 6;
  const int row = a.first_row + static_cast<int>(blockIdx.x) * kRows + (kRows == 1 ? 0 : wave);
  int rows = a.num_rows;
  if (a.row_limit != nullptr && *a.row_limit < rows) rows = *a.row_limit;
  if (row >= rows) return;  // the same for every thread that meets the barriers below

  const vec16* x = a.x + static_cast<size_t>(row) * a.x_row_vecs;
  const vec16* residual = kNorm && a.residual != nullptr ? a.residual + static_cast<size_t>(row) * a.residual_row_vecs : nullptr;
  float y[kVecs][8];
  float sum = 0.0f;
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    const int v = t + u * kRowThreads;
    if (v < a.row_vecs) {
      unpack8(__builtin_nontemporal_load(x + v), y[u]);  // read once: not worth the cache it would take
      if (kNorm && residual != nullptr) {
        float r[8];
        unpack8(__builtin_nontemporal_load(residual + v), r);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[u][i] += r[i];
        if (a.residual_out != nullptr) a.residual_out[static_cast<size_t>(row) * a.row_vecs + v] = pack8(y[u]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[u][i] = 0.0f;
    }
    if constexpr (kNorm) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(y[u][i], y[u][i], sum);
    }
  }
  if constexpr (kNorm) {
    sum = row_sum<kWaves>(sum, sums, wave);
    float mean = sum / static_cast<float>(a.row_vecs * 8) + a.eps;
    // Below, squares under the least fp32 value, 2^-149, would count for something (each loses up to 2^-150); above, the
    // sum has overflowed.  Then the row is divided by a power of two first.  The same for every thread of the row.
    if (__builtin_expect(!(mean >= 0x1p-120f && mean <= 0x1.fffffep127f), 0)) {
      uint32_t largest = 0;
#pragma unroll
      for (int u = 0; u < kVecs; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = umax(largest, __float_as_uint(y[u][i]) & 0x7fffffffu);
      largest = row_max<kWaves>(largest, maxima, wave);
      // A row that holds an infinity or a NaN, or nothing but zeros, is left as it is.
      if (largest != 0 && largest < 0x7f800000u) {
        // Of the row's largest magnitude and of epsilon's root, whichever is larger is brought near one.
        int exponent = __builtin_amdgcn_frexp_expf(__uint_as_float(largest));
        if (a.eps > 0.0f) {
          const int root = __builtin_amdgcn_frexp_expf(a.eps) >> 1;
          exponent = exponent > root ? exponent : root;
        }
        sum = 0.0f;
#pragma unroll
        for (int u = 0; u < kVecs; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[u][i] = __builtin_amdgcn_ldexpf(y[u][i], -exponent);
            sum = __builtin_fmaf(y[u][i], y[u][i], sum);
          }
        sum = row_sum<kWaves>(sum, sums, wave);
        mean = sum / static_cast<float>(a.row_vecs * 8) + __builtin_amdgcn_ldexpf(a.eps, -2 * exponent);
      }
      if constexpr (kWaves > 1) __syncthreads();  // `maxima` and `sums` have been read
    }
    const float inv = 1.0f / sqrtf(mean);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = t + u * kRowThreads;
      if (v < a.row_vecs) {
        float w[8];
        unpack8(a.weight[v], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[u][i] = y[u][i] * inv * w[i];
        if (a.normed != nullptr) a.normed[static_cast<size_t>(row) * a.row_vecs + v] = pack8(y[u]);
      }
    }
  }

  uint32_t amax[kVecs];
#pragma unroll
  for (int u = 0; u < kVecs; ++u) {
    amax[u] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax[u] = umax(amax[u], __float_as_uint(y[u][i]) & 0x7fffffffu);
  }
  uint2* q = a.q + static_cast<size_t>(row) * a.row_vecs;
  float* scales = a.scales + static_cast<size_t>(row) * a.scales_row_stride;
  if constexpr (kFormat == kQuantInt8) {
    uint32_t m = amax[0];
#pragma unroll
    for (int u = 1; u < kVecs; ++u) m = umax(m, amax[u]);
    m = row_max<kWaves>(m, maxima, wave);
    // One value for the whole row: in a scalar register the range test costs no vector instruction.
    const float scale = wave_read(scale_of<kFormat>(m), 0);
    if (t == 0) *scales = scale;
    const Divisor divide(scale);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = t + u * kRowThreads;
      if (v < a.row_vecs) store_codes<kNorm>(q + v, quantize8<kFormat>(y[u], divide));
    }
  } else {
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = t + u * kRowThreads;
      const float scale = scale_of<kFormat>(block_max(amax[u]));  // every lane takes part
      if (v < a.row_vecs) {
        if (v % kQuantBlockLanes == 0) scales[static_cast<size_t>(v / kQuantBlockLanes) * a.scales_hidden_stride] = scale;
        store_codes<kNorm>(q + v, quantize8<kFormat>(y[u], Divisor(scale)));
      }
    }
  }
}

template <int kFormat>
__global__ __launch_bounds__(256) void ep_dequantize_rows_kernel(const DequantizeArgs a) {
  int rows = a.num_rows;
  if (a.row_limit != nullptr && *a.row_limit < rows) rows = *a.row_limit;
  const long long total = static_cast<long long>(rows) * a.row_vecs;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * 256) {
    const int row = static_cast<int>(i / a.row_vecs);
    const int v = static_cast<int>(i - static_cast<long long>(row) * a.row_vecs);
    const float scale = a.scales[static_cast<size_t>(row) * a.scales_row_stride +
                                 (kFormat == kQuantInt8 ? 0 : static_cast<size_t>(v / kQuantBlockLanes) * a.scales_hidden_stride)];
    const uint2 q = a.q[i];
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t word = j < 4 ? q.x : q.y;
      if constexpr (kFormat == kQuantInt8) {
        f[j] = static_cast<float>(static_cast<int>(word << (24 - 8 * (j & 3))) >> 24);
      } else {
        switch (j & 3) {  // the byte is part of the instruction
          case 0: f[j] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 0); break;
          case 1: f[j] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 1); break;
          case 2: f[j] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 2); break;
          default: f[j] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(word), 3); break;
        }
      }
      f[j] *= scale;
    }
    if (a.stream_output) __builtin_nontemporal_store(pack8(f), a.out + i);
    else a.out[i] = pack8(f);
  }
}

template <bool kNorm, int kFormat>
hipError_t launch_quantize_as(const QuantizeArgs& args, hipStream_t stream) {
  // A launch has fewer than 2^32 threads: very many rows take several.
  const auto in_pieces = [&](auto kernel, int rows_at_once, int threads, int rows_per_group) {
    QuantizeArgs a = args;
    for (long long first = 0; first < args.num_rows; first += rows_at_once) {
      const long long left = args.num_rows - first;
      const long long rows = left < rows_at_once ? left : rows_at_once;
      a.first_row = static_cast<int>(first);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((rows + rows_per_group - 1) / rows_per_group)), dim3(threads), 0,
                         stream, a);
    }
  };
  const auto wave_rows = [&](auto kernel) { in_pieces(kernel, 1 << 25, 4 * kWave, 4); };
  const auto wide_rows = [&](auto kernel, int threads) { in_pieces(kernel, 1 << 21, threads, 1); };
  const QuantizeArgs& a = args;
  // With fewer rows than compute units the latency of one row is the time: more threads to a row, fewer vectors each
  // (16 rows of 7168 columns: 6.6 us with 256 threads of four vectors, 4.8 us with 1024 of one).  Measured and taken for these
  // widths only: 16 rows of 4096, a wave each, take 7.5 us.
  if (a.num_rows <= 256 && a.row_vecs > 512 && a.row_vecs <= 1024) wide_rows(&ep_quantize_rows_kernel<1024, 1, kNorm, kFormat>, 1024);
  else if (a.row_vecs <= 64) wave_rows(&ep_quantize_rows_kernel<64, 1, kNorm, kFormat>);
  else if (a.row_vecs <= 128) wave_rows(&ep_quantize_rows_kernel<64, 2, kNorm, kFormat>);
  else if (a.row_vecs <= 256) wave_rows(&ep_quantize_rows_kernel<64, 4, kNorm, kFormat>);
  else if (a.row_vecs <= 512) wave_rows(&ep_quantize_rows_kernel<64, 8, kNorm, kFormat>);
  else if (a.row_vecs <= 1024) wide_rows(&ep_quantize_rows_kernel<256, 4, kNorm, kFormat>, 256);
  else if (a.row_vecs <= 2048) wide_rows(&ep_quantize_rows_kernel<512, 4, kNorm, kFormat>, 512);
  else if (a.row_vecs <= 4096) wide_rows(&ep_quantize_rows_kernel<1024, 4, kNorm, kFormat>, 1024);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_rows(const QuantizeArgs& a, int format, hipStream_t stream) {
  if (a.num_rows == 0) return hipSuccess;
  const bool norm = a.weight != nullptr;
  if (format == kQuantInt8)
    return norm ? launch_quantize_as<true, kQuantInt8>(a, stream) : launch_quantize_as<false, kQuantInt8>(a, stream);
  return norm ? launch_quantize_as<true, kQuantE4m3>(a, stream) : launch_quantize_as<false, kQuantE4m3>(a, stream);
}

hipError_t launch_dequantize_rows(const DequantizeArgs& args, int format, hipStream_t stream) {
  if (args.num_rows == 0) return hipSuccess;
  DequantizeArgs a = args;
  // An output of a good part of the memory-side cache's size goes straight to HBM: what it would push out of that
  // cache (the codes themselves, the norm's other outputs) is read again sooner than its first rows.  Quantising
  // and reading back 65536 x 2048: 141 us with the store left to the caches, 124 us; norm and reading back 8192 x
  // 7168: 103 and 99 us.
  a.stream_output = static_cast<long long>(a.num_rows) * a.row_vecs * 16 >= (64ll << 20);
  const long long units = static_cast<long long>(a.num_rows) * a.row_vecs;
  const long long blocks = (units + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks < 16384 ? blocks : 16384));
  if (format == kQuantInt8)
    hipLaunchKernelGGL((ep_dequantize_rows_kernel<kQuantInt8>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((ep_dequantize_rows_kernel<kQuantE4m3>), grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mi_ep
