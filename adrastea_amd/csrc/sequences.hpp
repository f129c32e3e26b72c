// What the kernels for several packed sequences share: their arguments, and the search for a row's sequence.
#pragma once

#include "adr_common.hpp"

namespace adr {

// (x, y, z, page) strides of key and value pages, or of packed keys and values (page unused), in elements
struct KvStrides {
  int64_t x, y, z, p;
};

struct RotaryArgs {
  half_t* q_out;
  const half_t* q;    // null: keys and values only
  int so_x, so_y, so_z, sq_x, sq_y, sq_z;
  const half_t* k;    // null: queries only (adr_rotary_f16)
  const half_t* v;
  int sk_x, sk_y, sk_z, sv_x, sv_y, sv_z;
  const int* positions;  // null: positions in the cache
  const double* turns;
  int dims, pairs;       // pairs: ADR_ROTARY_PAIRS
  float magnitude;
  int heads, kv_heads, rows, d;
  adr_paged_cache cache;
  adr_paged_batch batch;
};
hipError_t launch_rotary(hipStream_t stream, const RotaryArgs& a);

// Rows are drafted tokens, and the last keys of their sequence: a row sees all keys before those, and of those what its bits say.
constexpr uint32_t MASK_TREE = 2;

constexpr int MOST_KEYS = 1 << 30;  // of a sequence (a workgroup's tiles beyond the last key still count in 31 bits)

// Attention of packed rows over pages or packed keys (table null).
struct SequencesArgs {
  half_t* out;
  const half_t* q;
  const half_t* k;
  const half_t* v;
  int so_x, so_y, so_z, sq_x, sq_y, sq_z;
  KvStrides sk, sv;
  const int* row_offsets;
  const int* keys_of;  // pages: lengths [sequences]; packed: key offsets [sequences + 1]
  const int* table;
  int sequences, rows, keys;  // keys: of the packed tensor
  int heads, kv_heads, group, d;
  int table_width, table_pitch, pages, page_size;
  int longest_rows, longest;
  float c;             // scale * log2(e) / temperature
  uint32_t mask;
  // In 8 bits: k and v are codes, and these their scales (y slot, z head, p page); null: k and v are fp16.
  const half_t* k_scale;
  const half_t* v_scale;
  KvStrides sks, svs;
  const int* tree;     // MASK_TREE: [rows, tree_words] bits of the drafted tokens that a row sees
  int tree_words, tree_pitch;
};
// Which kernel, and how the keys are shared over workgroups (attention_sequences.hip).
struct SequencesPlan {
  enum Kind { ANY_LAYOUT, FEW_ROWS, TILES } kind;
  int waves;  // wavefronts of a workgroup
  int parts;  // workgroups of each key head that share all its work; 0: one for each block of rows
  int shift;  // log2 of the key tiles of a piece of the work
  int least;  // pieces that each workgroup has at least
  int64_t workspace_bytes;
  bool longest_first = false;  // unshared blocks of few rows: the sequences with the most keys first
};
SequencesPlan sequences_plan(const SequencesArgs& a, int cus, int64_t avail);
hipError_t launch_attention_sequences(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p,
                                      void* workspace);
// The same where keys and values are codes (attention_u8.hip).
SequencesPlan sequences_u8_plan(const SequencesArgs& a, int cus, int64_t avail);
hipError_t launch_attention_u8(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace);


// The last of `sequences` whose first row is not behind `row`, by all lanes of a wavefront: 64 offsets a
// step, each a trip to memory, so that 4096 sequences take two.  (Of several at one offset the last: the others
// are empty.)  Without one the result is 0, and the caller finds the row outside of it.
__device__ __forceinline__ int sequence_of_row(const int* __restrict__ offsets, int sequences, int row, int lane) {
  int lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int at = lo + lane * step;
    const bool in = at < hi && offsets[at] <= row;
    const int n = __popcll(__ballot(in));
    if (n == 0) return 0;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

__device__ __forceinline__ int clamp_to(int v, int high) { return min(max(v, 0), high); }

}  // namespace adr
