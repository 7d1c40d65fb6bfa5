// fk_prefix.h -- what fk_prefix.cu needs of fk_decode.cu: the own-tokens part
// of a shared-prefix decode, run by the paged decode kernel with its segments'
// (max, sum, acc) left in the workspace for the join.
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
// The records it leaves: those of item i are i + info[i].x .. (info[i].y of
// them), each `slots` query-head slots of HEAD_DIM floats.
struct OwnRecords {
  const float2* ml;
  const float* acc;
  const int2* info;
  int hp, qc, slots, per_seq;  // KV heads of an item, query chunks of a KV head, slots, items of a sequence
  int ctas;                    // of the own part's grid: an item has at most one record in each
  // The records of item i.  Where a wait of the own part ran out, info[i] may
  // never have been written: it is then what the scratch held, and taken only if
  // it names records that exist.
  __device__ int2 of(long long i) const {
    const int2 r = __ldcg(info + i);
    return r.x >= 0 && r.y >= 0 && r.x <= ctas - r.y ? r : make_int2(0, 0);
  }
  // Item (within its sequence) and slot of query head g of KV head h's group.
  __device__ void find(int h, int g, int* item, int* slot) const {
    if (qc == 1) {
      *item = h / hp;
      *slot = (h % hp) * GPAD + g;
    } else {
      const int c = g >> 3;
      *item = hp == 2 ? h * ((qc + 1) >> 1) + (c >> 1) : h * qc + c;
      *slot = (hp == 2 ? (c & 1) * GPAD : 0) + (g & 7);
    }
  }
};
// Nothing in its workspace need be set before.  *ticket is ticket_value from
// when the kernel has waited for what precedes it in the stream.
int own_part_launch(OwnPart& own, int2* info, unsigned long long* ticket, unsigned long long ticket_value, int* status, size_t ws_bytes, cudaStream_t stream, OwnRecords* records);
// A tensor map with 128-byte swizzle (fk_decode.cu).
int encode_map(CUtensorMap* map, int kv, int rank, const void* base, const uint64_t* dims, const uint64_t* strides_b,
               const uint32_t* box);
// fk_debug_configure's settings.
void debug_settings(unsigned long long* wait_ns, int* inject);

}  // namespace fk
