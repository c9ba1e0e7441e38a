// Launch interface of the appends of rows to KV caches and the reads back
// (kv_append.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rotary.h"

namespace qm {

constexpr uint32_t kMaxAppendSeqs = 32;  // sequences a launch (kernel-argument table)

// The pages of one cache: k, v, ks, vs of a Q8 cache, or k alone (blocks) of a
// 4-bit one.
struct KvPages {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int32_t* pt;
};

struct KvAppendSeq {
  KvPages p;
  uint32_t start;       // cache position of the sequence's first new row
  uint32_t rows;
  uint32_t row0;        // that row's index in the call
  uint32_t unit_begin;  // first workgroup; filled by the launcher
  int32_t new_page_first;  // first logical page that the call materialises
  int32_t new_page_count;
  int32_t new_page_id;     // its physical id (ids are consecutive)
};

struct KvAppendArgs {
  double freq[kRotaryMaxDim / 2];  // radians per position
  KvAppendSeq seqs[kMaxAppendSeqs];
  const void* k;  // bf16 rows of kv_heads heads of head_dim (fp32 in launch_q4kv_append_f32)
  const void* v;
  uint64_t k_stride, v_stride;  // elements between rows
  const uint32_t* positions;    // of every row of the call, or null: the row's place in its cache
  RotaryTensor q;               // queries to rotate; in == null: none
  float factor;                 // of sine and cosine
  uint32_t n_seqs;
  uint32_t kv_heads;
  uint32_t head_dim;
  uint32_t head_dim_pad;
  uint32_t rotary_dim;  // 0: keys as given
  uint32_t offset;      // first rotated element of a key
  uint32_t half_log;    // least with 2^half_log >= rotary_dim / 2; filled by the launcher
  uint32_t row0, rows;  // the launch's rows of the call; filled by the launcher
  uint32_t units;       // workgroups that append; filled by the launcher
  uint32_t share;       // KV heads of one such workgroup; filled by the launcher
  uint32_t q_items;     // filled by the launcher
  uint32_t q_groups;
};

// Workgroups that a launch takes: its threads are counted in 32 bits.
constexpr uint64_t kv_append_most(uint32_t head_dim_pad) { return 0xFFFFFFFFull / (4 * head_dim_pad); }
constexpr uint64_t kv_load_most(uint32_t head_dim_pad) { return 0xFFFFFFFFull / (5 * head_dim_pad / 2); }
// Workgroups that rotate queries share a row where rows are few, up to this many in all.
constexpr uint32_t kQueryGroups = 1024;

// `vec`: keys and values take 8-byte loads (4 elements) and a key's pairs lie 4
// elements at a time; `qvec`: queries as launch_rotary's vec.
hipError_t launch_kv_append(const KvAppendArgs& a, uint32_t bits, bool interleaved, bool vec, bool qvec,
                            hipStream_t st);

// fp32 rows into 4-bit caches, as given (no rotation, no queries).  `vec`: rows
// take 16-byte loads.
hipError_t launch_q4kv_append_f32(const KvAppendArgs& a, bool vec, hipStream_t st);

struct KvLoadArgs {
  KvPages p;
  uint16_t* k;  // bf16 [count][kv_heads][head_dim], or null
  uint16_t* v;
  uint32_t first, count;
  uint32_t kv_heads;
  uint32_t head_dim;
  uint32_t head_dim_pad;
};
hipError_t launch_kv_load(const KvLoadArgs& a, uint32_t bits, hipStream_t st);

}  // namespace qm
