// Stages of rows in LDS, filled by loads that bypass the registers, for gfx950.
#pragma once
#include "ep_expert.h"

namespace mi_ep {

typedef int int4v __attribute__((ext_vector_type(4)));

constexpr int kStageK = 128;                             // bytes of k in a stage
constexpr int kChunkBytes = 1024;                        // what one load instruction of a wave moves
constexpr int kOutside = static_cast<int>(0x80000000u);  // an offset beyond every descriptor

// 64 lanes x 16 bytes from global memory to 1 KiB of LDS at `lds` (wave-uniform), not waited for.  In
// assembly because the compiler would wait for every load before the next LDS read of any address; the
// waits are written at the end of each step instead.  A lane whose offset lies outside the descriptor moves
// zeros and makes no memory request.  kStream (the streaming hint) is for weights that one tile of rows reads and
// nobody again: they pass the memory-side cache by, which keeps the products until the next operator reads them, and
// the memory does not turn round between reads and writes all the time.  256 experts of 64 rows x 4096 x 4096: 823 us with
// neither this nor the results written through into that cache, 788 with the first only, 698 with both; where tiles share
// their weights the hint costs (8192^3 435 us without, 474 with).
template <bool kStream = false>
__device__ __forceinline__ void load_to_lds(int4v descriptor, int lds, int lane_offset, int scalar_offset) {
  if constexpr (kStream)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen nt lds"
                 :
                 : "s"(lds), "v"(lane_offset), "s"(descriptor), "s"(scalar_offset)
                 : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(lds), "v"(lane_offset), "s"(descriptor), "s"(scalar_offset)
                 : "memory");
}
__device__ __forceinline__ void load_word_to_lds(int4v descriptor, int lds, int lane_offset) {  // 4 bytes a lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(lane_offset), "s"(descriptor)
               : "memory");
}
__device__ __forceinline__ int4v descriptor_of(const void* base, int bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  return int4v{__builtin_amdgcn_readfirstlane(static_cast<int>(at)),
               __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32) & 0xffff), __builtin_amdgcn_readfirstlane(bytes),
               kRawBufferFormat};
}

// The byte address in LDS of a pointer into it.
__device__ __forceinline__ int lds_address(const unsigned char* p) {
  return static_cast<int>((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p);
}

// A lane's part in the loads and reads of a stage.  A stage holds rows of 128 bytes, whole cache lines (of half lines
// the memory delivers a fifth less); the eight 16-byte pieces of a row are permuted by exclusive or with half its
// number, so that 16 lanes reading one piece of 16 rows meet all 64 banks.  A load instruction fills eight rows in
// order; lane l of it fetches the piece that belongs at l, which in every other eight rows is the one 64 bytes away.
struct Place {
  int piece, row, read_at;
  __device__ __forceinline__ explicit Place(int lane) {
    const int r = lane & 31;
    piece = ((lane & 7) ^ (lane >> 4)) * 16;
    row = lane >> 3;
    read_at = r * 128 + (((lane >> 5) ^ ((r >> 1) & 7)) * 16);
  }
  __device__ __forceinline__ int piece_of(int eight) const { return piece ^ ((eight & 1) * 64); }
};

}  // namespace mi_ep
