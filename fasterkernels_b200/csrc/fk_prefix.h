// fk_prefix.h -- what fk_prefix.cu needs of fk_decode.cu: the own-tokens part
// of a shared-prefix decode, run by the paged decode kernel with its running
// (max, sum, acc) stored instead of an output.
#pragma once
#include <mutex>

#include "fk_decode_kernel.cuh"

namespace fk {

struct OwnPart {
  Params p;
  int kv, device, q_al16;
};

// Argument checks and tensor maps (FK_OK, or an error).
int own_part_prepare(OwnPart* own, const fk_prefix_args& a, void* workspace, int* device);
// Leading 32-bit words of its workspace that must be zero before the launch.
int own_part_zero_words(const OwnPart& own, size_t ws_bytes);
int own_part_launch(OwnPart& own, float2* ml, float* acc, size_t ws_bytes, cudaStream_t stream);
// A tensor map with 128-byte swizzle (fk_decode.cu).
int encode_map(CUtensorMap* map, int kv, int rank, const void* base, const uint64_t* dims, const uint64_t* strides_b,
               const uint32_t* box);
// fk_debug_configure's settings.
void debug_settings(unsigned long long* wait_ns, int* inject);

}  // namespace fk
