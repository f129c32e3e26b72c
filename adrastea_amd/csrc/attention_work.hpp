// What the kernels of attention over several sequences share: their job, who does which part of it, the row that a
// wavefront computes by itself, and the launch that adds up the parts of a block.
#pragma once

#include <math.h>

#include "attention_parts.hpp"
#include "sequences.hpp"

namespace adr {
namespace {

// Below any score of finite operands (256 * 65504^2 < 2^41, times at most 2^58 log2(e)); exp2(-inf - NO_SCORE) is 0, not NaN.
constexpr float NO_SCORE = -1.0e30f;

// A row's probabilities are 2^(s c - R), rounded to fp16 for the second product.  R follows the largest s c that was seen: 7 below it
// where it moves, and it moves, with the sums rescaled, when that has grown to more than 15 above, which after the first tiles is
// rare.  So the largest probability is 2^7 to 2^15 (65504 is fp16's largest number), and one of 2^-14 is still as exact
// as 1 is; below, the error of 2^-25 is 2^-32 of the largest, and keys that weigh as little are lost altogether.  (With R up
// to 8 below, each of 6000 keys that weigh 2^-25.5 was lost: 2^-13 of the result.)
constexpr float BELOW = 7.0f, GROWN = 15.0f;
// s c - R is one fma, exact but for its last step, but the largest s c is itself rounded: at 2^31 by up to 2^7, so that the
// largest probability could be 2^128 or 2^-128.  A step above what was found, it is no smaller than it should be at least, and no
// probability or sum is infinite that should not be; rows whose R is beyond FAR_SCORE in the end, where it can be larger by
// more than 2, are computed again by row_by_wave.  (An infinite one has made the row NaN, as it should be.)
constexpr float FAR_SCORE = 0x1p24f;
__device__ __forceinline__ bool is_far(float r) { return fabsf(r) > FAR_SCORE && fabsf(r) < INFINITY; }
__device__ __forceinline__ float above(float top) { return fmaf(fabsf(top), 0x1p-23f, top); }

// A weighted mean of values, rounded to fp16.  Its weights are off by up to 2^-11 each (fp16 in the second product, 32 bits in their
// sum), so that a mean of values near the largest number of fp16 can lie as far beyond it, and would be rounded to
// infinity: it is that number.
constexpr float LARGEST = 65504.0f;
__device__ __forceinline__ half_t mean_of(float v) {
  return (half_t)(fabsf(v) < LARGEST * 1.01f ? __builtin_amdgcn_fmed3f(v, -LARGEST, LARGEST) : v);
}
// Four of them; false: not all are finite.  (One that is rounded to infinity is rare, and looked at again.)
__device__ __forceinline__ bool round_means(half4_t& h, const float4_t& v, float factor) {
  bool finite = true;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    h[j] = (half_t)(v[j] * factor);
    finite = finite && fabsf((float)h[j]) < INFINITY;
  }
  if (finite) return true;
  finite = true;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    h[j] = mean_of(v[j] * factor);
    finite = finite && fabsf((float)h[j]) < INFINITY;
  }
  return finite;
}

// Eight codes c as c 2^-24.
__device__ __forceinline__ half8_t widened(uint32_t w0, uint32_t w1) {
  const u32x4_t r = {__builtin_amdgcn_perm(0u, w0, 0x0c010c00u), __builtin_amdgcn_perm(0u, w0, 0x0c030c02u),
                     __builtin_amdgcn_perm(0u, w1, 0x0c010c00u), __builtin_amdgcn_perm(0u, w1, 0x0c030c02u)};
  return __builtin_bit_cast(half8_t, r);
}
constexpr float WIDENED = 0x1p-24f;

// The largest probability times scale may be this much above the reference, in log2 units.
constexpr float GROWN_U8 = GROWN - 0.5f;

// What a kernel is given.  Share of the work: see below.
struct Job : SequencesArgs {
  int page_shift;   // log2 of the slots of a page (16 at least: 16 keys from a multiple of 16 on lie on one page)
  int parts;        // workgroups of a key head that share its work; 0: unshared
  int shift;        // few rows: log2 of a piece's tiles
  int least;        // pieces (many rows: tiles) that a workgroup has at least
  double per_head;  // 1 / group
  float* part_o;    // [slot][key head][ROWS][HD] unnormalised sums
  float2* part_ml;  // [slot][key head][ROWS] (maximum in log2 units, sum)
  struct Seam* seams;  // [parts][key head], of many rows half as many
  int longest_first;   // Roster's sequences in the order of their keys
};

// The job is read where it is used, by scalar loads from the kernel's arguments (of which it is the only one): kept in
// registers from the start, what only the end of a kernel needs would push out what its loops need -- 25 scalar registers
// were spilled into vector ones.  Loads do not move across arguments().
typedef const __attribute__((address_space(4))) Job& Args;
__device__ __forceinline__ Args arguments() {
  auto p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const __attribute__((address_space(4))) Job*)p;
}

// What the start of a block needs, or (ALL false) the division of the work, by one wait for all of it.
template <bool PAGED, bool ALL = true>
__device__ __forceinline__ void early(Args a) {
  if constexpr (!ALL && PAGED)
    asm volatile("" ::"s"(a.kv_heads), "s"(a.row_offsets), "s"(a.keys_of), "s"(a.rows), "s"(a.sequences), "s"(a.group),
                 "s"(a.parts), "s"(a.shift), "s"(a.least), "s"(a.table_width), "s"(a.page_size));
  else if constexpr (!ALL)
    asm volatile("" ::"s"(a.kv_heads), "s"(a.row_offsets), "s"(a.keys_of), "s"(a.rows), "s"(a.sequences), "s"(a.group),
                 "s"(a.parts), "s"(a.shift), "s"(a.least), "s"(a.keys));
  else if constexpr (PAGED)
    asm volatile("" ::"s"(a.kv_heads), "s"(a.row_offsets), "s"(a.keys_of), "s"(a.rows), "s"(a.sequences), "s"(a.group),
                 "s"(a.per_head), "s"(a.mask), "s"(a.d), "s"(a.q), "s"(a.sq_y), "s"(a.sq_z), "s"(a.k), "s"(a.v), "s"(a.sk.y),
                 "s"(a.sk.z), "s"(a.sv.y), "s"(a.sv.z), "s"(a.sk.p), "s"(a.sv.p), "s"(a.table), "s"(a.table_width),
                 "s"(a.page_size), "s"(a.table_pitch), "s"(a.pages), "s"(a.page_shift));
  else
    asm volatile("" ::"s"(a.kv_heads), "s"(a.row_offsets), "s"(a.keys_of), "s"(a.rows), "s"(a.sequences), "s"(a.group),
                 "s"(a.per_head), "s"(a.mask), "s"(a.d), "s"(a.q), "s"(a.sq_y), "s"(a.sq_z), "s"(a.k), "s"(a.v), "s"(a.sk.y),
                 "s"(a.sk.z), "s"(a.sv.y), "s"(a.sv.z), "s"(a.keys));
}

// A list row's row: the quotient is at least 0.5 / group away from the next integer, far more than the product's error.
__device__ __forceinline__ int row_of_list(Args a, int list_row) { return (int)(((double)list_row + 0.5) * a.per_head); }

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The thread's index, likewise: what a kernel derives from it for one block is not kept for the next.
__device__ __forceinline__ int thread_index() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A sequence's rows and keys.
struct Sequence {
  int index, row0, rows;  // first row of the [heads, rows, d] views
  int key0, keys;         // first key of packed ones
};

__device__ __forceinline__ Sequence sequence_at(Args a, int s, bool paged) {
  // (all four loads at once: one way to memory)
  const int r0 = a.row_offsets[s], r1 = a.row_offsets[s + 1], k0 = a.keys_of[s], k1 = a.keys_of[s + (paged ? 0 : 1)];
  Sequence q;
  q.index = s;
  q.row0 = clamp_to(r0, a.rows);
  q.rows = max(clamp_to(r1, a.rows) - q.row0, 0);
  if (paged) {
    const int64_t room = min((int64_t)a.table_width * a.page_size, (int64_t)MOST_KEYS);
    q.key0 = 0;
    q.keys = (int)min((int64_t)max(k0, 0), room);
  } else {
    q.key0 = clamp_to(k0, a.keys);
    q.keys = max(clamp_to(k1, a.keys) - q.key0, 0);
  }
  return q;
}

// Key x of the sequence as element offsets of its key and value rows (head 0); false: on no page of the cache.
__device__ __forceinline__ bool key_at(Args a, const Sequence& q, int x, int64_t& k, int64_t& v) {
  if (!a.table) {
    k = (q.key0 + (int64_t)x) * a.sk.y;
    v = (q.key0 + (int64_t)x) * a.sv.y;
    return true;
  }
  const int at = x / a.page_size, slot = x - at * a.page_size;
  const int page = a.table[(int64_t)q.index * a.table_pitch + at];
  const bool good = page >= 0 && page < a.pages;
  k = good ? page * a.sk.p + slot * a.sk.y : 0;
  v = good ? page * a.sv.p + slot * a.sv.y : 0;
  return good;
}

// MASK_TREE: which of 32 keys the row sees, from the rel-th drafted one on (what is negative is in front of the draft, and seen by
// all): two words of its bits, shifted.
__device__ __forceinline__ uint32_t tree_window(Args a, int64_t row, int rel) {
  const int word = rel >> 5;  // (rounds down)
  auto bits = [&](int w) __attribute__((always_inline)) -> uint32_t {
    return w < 0 ? ~0u : w < a.tree_words ? (uint32_t)a.tree[row * a.tree_pitch + w] : 0u;
  };
  return __builtin_amdgcn_alignbit(bits(word + 1), bits(word), rel & 31);
}

// One row of one query head by one wavefront, at any strides: 64 keys at a time, a lane to a key for the scores
// and a lane to every 64th column for the sums.  Only keys that the row sees are read.  Probabilities stay in 32 bits, and
// scores unscaled until their maximum is subtracted: right for scores of any size.  (Columns col0 ... col1 - 1 are stored.  Without
// TREE rows that see what is in front of them need fewer scalar registers of the kernels that end with this.)
constexpr int GENERAL_MAX_D = 256;
template <bool TREE = true>
__device__ __forceinline__ void row_by_wave(Args a, const Sequence& q, int j, int h, int lane, int col0 = 0, int col1 = GENERAL_MAX_D) {
  const int64_t row = (int64_t)q.row0 + j;
  const half_t* const Q = a.q + h * (int64_t)a.sq_z + row * a.sq_y;
  const half_t* const K = a.k + (h / a.group) * a.sk.z;
  const half_t* const V = a.v + (h / a.group) * a.sv.z;
  const int end = a.mask == ADR_MASK_CAUSAL ? min(q.keys, j + q.keys - q.rows + 1) : q.keys;  // (may be negative)
  float o[GENERAL_MAX_D / 64] = {}, m = NO_SCORE, l = 0.0f;
  for (int x0 = 0; x0 < end; x0 += 64) {
    const int x = x0 + lane;
    float s = -INFINITY;
    int64_t ko = 0, vo = 0;
    bool good = true;
    const bool seen = x < end && (!TREE || a.mask != MASK_TREE || (tree_window(a, row, x - (q.keys - q.rows)) & 1));
    if (seen) {
      good = key_at(a, q, x, ko, vo);
      s = 0.0f;
      if (good)
        for (int i = 0; i < a.d; i++) s = fmaf((float)Q[i * (int64_t)a.sq_x], (float)K[ko + i * a.sk.x], s);
      if (!good) s = NAN;
    }
    float top = s;
    for (int i = 32; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));  // (not the NaNs)
    const float m_new = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f((m - m_new) * a.c);
    m = m_new;
    const float p = __builtin_amdgcn_exp2f((s - m) * a.c);
    l = l * alpha + p;
#pragma unroll
    for (int c = 0; c < GENERAL_MAX_D / 64; c++) o[c] *= alpha;
    auto add = [&](int e) __attribute__((always_inline)) {
      const float pe = __shfl(p, e);
      const int64_t at = __shfl(vo, e);
      if (!__shfl((int)good, e)) {
#pragma unroll
        for (int c = 0; c < GENERAL_MAX_D / 64; c++) o[c] = NAN;
        return;
      }
#pragma unroll
      for (int c = 0; c < GENERAL_MAX_D / 64; c++)
        if (c * 64 + lane < a.d) o[c] = fmaf(pe, (float)V[at + (c * 64 + lane) * a.sv.x], o[c]);
    };
    if constexpr (TREE) {
      for (uint64_t left = __ballot(seen); left != 0; left &= left - 1) add(__builtin_ctzll(left));
    } else {
      const int n = min(64, end - x0);
      for (int e = 0; e < n; e++) add(e);
    }
  }
  for (int i = 32; i > 0; i >>= 1) l += __shfl_xor(l, i);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  half_t* const O = a.out + h * (int64_t)a.so_z + row * a.so_y;
#pragma unroll
  for (int c = 0; c < GENERAL_MAX_D / 64; c++)
    if (c * 64 + lane < a.d && c * 64 + lane >= col0 && c * 64 + lane < col1)
      O[(c * 64 + lane) * (int64_t)a.so_x] = mean_of(o[c] * inv);
}

// The same over codes.  A key counts as NaN where a scale of it is larger than those of the format, or no number.
__device__ __forceinline__ bool scale_fits(half_t s) { return fabsf((float)s) <= 513.5f; }

template <bool TREE = true>
__device__ __forceinline__ void row_by_wave_u8(Args a, const Sequence& q, int j, int h, int lane, int col0 = 0, int col1 = GENERAL_MAX_D) {
  const int64_t row = (int64_t)q.row0 + j;
  const int hk = h / a.group;
  const half_t* const Q = a.q + h * (int64_t)a.sq_z + row * a.sq_y;
  const uint8_t* const K = (const uint8_t*)a.k + hk * a.sk.z;
  const uint8_t* const V = (const uint8_t*)a.v + hk * a.sv.z;
  const int end = a.mask == ADR_MASK_CAUSAL ? min(q.keys, j + q.keys - q.rows + 1) : q.keys;  // (may be negative)
  float o[GENERAL_MAX_D / 64] = {}, m = NO_SCORE, l = 0.0f;
  for (int x0 = 0; x0 < end; x0 += 64) {
    const int x = x0 + lane;
    float s = -INFINITY, value_scale = 0.0f;
    int64_t vo = 0;
    const bool seen = x < end && (!TREE || a.mask != MASK_TREE || (tree_window(a, row, x - (q.keys - q.rows)) & 1));
    bool good = false;
    if (seen) {
      const int at = x / a.page_size, slot = x - at * a.page_size;
      const int page = a.table[(int64_t)q.index * a.table_pitch + at];
      s = NAN;
      if (page >= 0 && page < a.pages) {
        const half_t ks = a.k_scale[page * a.sks.p + slot * a.sks.y + hk * a.sks.z];
        const half_t vs = a.v_scale[page * a.svs.p + slot * a.svs.y + hk * a.svs.z];
        good = scale_fits(ks) && scale_fits(vs);
        if (good) {
          const int64_t ko = page * a.sk.p + slot * a.sk.y;
          float sum = 0.0f, none = 0.0f;
          for (int i = 0; i < a.d; i++) {
            const float qi = (float)Q[i * (int64_t)a.sq_x];
            sum = fmaf(qi, (float)K[ko + i * a.sk.x] - 127.5f, sum);
            none = fmaf(qi, 0.0f, none);
          }
          s = fmaf(sum, (float)ks, none);
          vo = page * a.sv.p + slot * a.sv.y;
          value_scale = (float)vs;
        }
      }
    }
    float top = s;
    for (int i = 32; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));  // (not the NaNs)
    const float m_new = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f((m - m_new) * a.c);
    m = m_new;
    const float p = __builtin_amdgcn_exp2f((s - m) * a.c);
    l = l * alpha + p;
#pragma unroll
    for (int c = 0; c < GENERAL_MAX_D / 64; c++) o[c] *= alpha;
    const int n = min(64, end - x0);
    for (int e = 0; e < n; e++) {
      if (!__shfl((int)good, e)) continue;
      const float pe = __shfl(p * value_scale, e);
      const int64_t at = __shfl(vo, e);
#pragma unroll
      for (int c = 0; c < GENERAL_MAX_D / 64; c++)
        if (c * 64 + lane < a.d) o[c] = fmaf(pe, (float)V[at + (c * 64 + lane) * a.sv.x] - 127.5f, o[c]);
    }
  }
  for (int i = 32; i > 0; i >>= 1) l += __shfl_xor(l, i);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  half_t* const O = a.out + h * (int64_t)a.so_z + row * a.so_y;
#pragma unroll
  for (int c = 0; c < GENERAL_MAX_D / 64; c++)
    if (c * 64 + lane < a.d && c * 64 + lane >= col0 && c * 64 + lane < col1)
      O[(c * 64 + lane) * (int64_t)a.so_x] = mean_of(o[c] * inv);
}

// Any layout: a wavefront per row and query head.
template <bool U8>
__device__ __forceinline__ void rows_one_by_one(Args a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i = (int64_t)blockIdx.x * 4 + wave; i < (int64_t)a.rows * a.heads; i += (int64_t)gridDim.x * 4) {
    const int h = (int)(i / a.rows), row = (int)(i - (int64_t)h * a.rows);
    const Sequence q = sequence_at(a, sequence_of_row(a.row_offsets, a.sequences, row, lane), a.table != nullptr);
    if (row < q.row0 || row >= q.row0 + q.rows) continue;
    if constexpr (U8) row_by_wave_u8(a, q, row - q.row0, h, lane);
    else row_by_wave(a, q, row - q.row0, h, lane);
  }
}

// ---- who does what -----------------------------------------------------------------------------------
//
// The rows of a sequence times the query heads of a group, R = rows * group, are one list (row of the sequence
// first, head of the group second), cut into blocks of ROWS: the heads of a group share every key that is read.
// The host knows neither the sequences' rows nor their keys, so the work is divided on the device, by every wavefront
// for itself and with the same result.  Unshared: a workgroup takes one block of one key head.  Shared: all blocks' keys
// are one line of pieces of 2^shift tiles, block after block, and each of `parts` workgroups of a key head takes the
// same length of it: no sequence, however long among short ones, holds up the others, and a workgroup has its
// start-up once.  A block that lies in one workgroup's stretch is finished there.  Of the others, a workgroup has at
// most the first and the last in its stretch; their results go to its two slots of the workspace, and are joined by a
// second launch, in order.
struct Line {
  int total, parts, shift;  // pieces, workgroups that have some, log2 of a piece's tiles
  // (exact: the product has fewer than 53 bits, and a quotient that is no integer lies too far below the next one)
  __device__ __forceinline__ int at(int part) const { return uniform((int)((double)total * (double)part / (double)parts)); }
};

// What the second launch needs of a divided block: of few rows, at the place where a stretch begins inside a block and no
// stretch before begins inside the same one.
struct Seam {
  int parts, slot;  // 0 parts: nothing to do here
  Sequence q;
  int block;
};

struct Block {
  Sequence q;
  int block;           // of the sequence's list
  int offset, pieces;  // of the block: where on the line the asked place lies in it, and all
};

__device__ __forceinline__ int add_scan(int v) {  // inclusive, over the lanes of a wavefront
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}

__device__ __forceinline__ int min_of_all(int v) {
  constexpr int NONE = 0x7fffffff;
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x112, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x114, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x118, 0xf, 0xf, false));
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  v = min(v, __builtin_amdgcn_update_dpp(NONE, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
  return __builtin_amdgcn_readlane(v, 63);
}

// Rows of a block, keys of a tile, log2 of the tiles of a piece
constexpr int FEW = 16, FEW_KEYS = 32, FEW_SHIFT = 2;
constexpr int MANY = 128, MANY_KEYS = 64;

// The sequences on the line, 256 at a time: lane l has sequences base + 64 e + l, read from memory once for the whole
// division where there are no more.
//
// ORDERED, where the job asks for it and there are at most 64: the sequences with the most keys come first.  Unshared blocks that are
// more than the compute units start in this order, and no long one is the last (64 sequences of 3 to 4000 keys over codes, 512
// blocks: the units were busy 63 % of the time).
template <int ROWS, int KEYS, bool PAGED, bool SHARED, bool ORDERED = false>
struct Roster {
  static constexpr int EACH = 4;
  typedef int each_t __attribute__((ext_vector_type(EACH)));
  each_t row0, rows, key0, keys;
  each_t upto;            // where on the line the sequence ends
  int which;              // ORDERED: lane l's sequence
  int base, before, end;  // first sequence, and the part of the line that these are

  static __device__ __forceinline__ int blocks_of(Args a, int rows) {
    return (int)(((int64_t)rows * a.group + ROWS - 1) / ROWS);
  }
  // A block's pieces: one at least, so that rows without keys are somebody's.
  static __device__ __forceinline__ int pieces_of(int keys, int shift) {
    return SHARED ? max(1, (((keys + KEYS - 1) / KEYS) + (1 << shift) - 1) >> shift) : 1;
  }
  __device__ __forceinline__ void load(Args a, int shift, int lane, int first, int line) {
    base = first;
    before = end = line;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      row0[e] = rows[e] = key0[e] = keys[e] = 0;
      if (base + 64 * e < a.sequences && base + 64 * e + lane < a.sequences) {
        const Sequence q = sequence_at(a, base + 64 * e + lane, PAGED);
        row0[e] = q.row0, rows[e] = q.rows, key0[e] = q.key0, keys[e] = q.keys;
      }
    }
    if constexpr (ORDERED) {
      which = lane;
      if (a.longest_first && a.sequences <= 64) {
        // (one number for each: its keys, then its place)
        const int n = a.sequences, size = min(keys[0], 1 << 24) * 64 + 63 - lane;
        int rank = 0;
        for (int i = 0; i < n; i++) rank += __builtin_amdgcn_readlane(size, i) > size;
        rank = 4 * (lane < n ? rank : lane);
        auto moved = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_ds_permute(rank, v); };
        which = moved(lane);
        row0[0] = moved(row0[0]), rows[0] = moved(rows[0]), key0[0] = moved(key0[0]), keys[0] = moved(keys[0]);
      }
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      upto[e] = end;
      if (base + 64 * e < a.sequences) {
        upto[e] += add_scan(blocks_of(a, rows[e]) * pieces_of(keys[e], shift));
        end = __builtin_amdgcn_readlane(upto[e], 63);
      }
    }
  }
  // The whole line.
  __device__ __forceinline__ Line line_of(Args a, int lane) {
    load(a, a.shift, lane, 0, 0);
    while (base + 64 * EACH < a.sequences) load(a, a.shift, lane, base + 64 * EACH, end);
    Line line = {end, max(1, end), a.shift};
    if (SHARED) line.parts = max(1, min(a.parts, end / a.least));
    return line;
  }
  // The block at `place` of the line; false: the line ends before (or offsets that decrease made it longer than it counts).
  __device__ __forceinline__ bool block_at(Args a, int shift, int place, int lane, Block& b) {
    if (place < before) load(a, shift, lane, 0, 0);
    while (place >= end) {
      if (base + 64 * EACH >= a.sequences) return false;
      load(a, shift, lane, base + 64 * EACH, end);
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const uint64_t behind = __ballot(upto[e] > place);
      if (behind) {
        const int at = __builtin_ctzll(behind);
        b.q = {ORDERED && e == 0 && base == 0 ? __builtin_amdgcn_readlane(which, at) : base + 64 * e + at, __builtin_amdgcn_readlane(row0[e], at), __builtin_amdgcn_readlane(rows[e], at),
               __builtin_amdgcn_readlane(key0[e], at), __builtin_amdgcn_readlane(keys[e], at)};
        const int blocks = blocks_of(a, b.q.rows), p = pieces_of(b.q.keys, shift);
        const int in = place - (__builtin_amdgcn_readlane(upto[e], at) - blocks * p);
        // (the last blocks first: under the mask they have the most keys)
        const int i = SHARED ? uniform(in / p) : in;
        b.block = blocks - 1 - i;
        b.offset = in - i * p;
        b.pieces = p;
        return in >= 0 && b.block >= 0;
      }
    }
    return false;
  }
};

// The seam at the beginning of stretch `part`, which lies in block b.
__device__ __forceinline__ Seam seam_at(const Line& line, int part, int place, const Block& b) {
  Seam s = {0, 0, b.q, b.block};
  if (part == 0 || b.offset == 0) return s;
  const int begin = place - b.offset, before = line.at(part - 1);
  if (before > begin) return s;
  // stretches part - 1 ... last; the first of them has the block behind others, unless it begins with it
  const int last = uniform((int)(((double)(begin + b.pieces) * (double)line.parts - 1.0) / (double)line.total));
  s.parts = min(last, line.parts - 1) - part + 2;
  s.slot = 2 * (part - 1) + (before != begin);
  return s;
}

// The share of a workgroup of the kernel for many rows.
struct Part {
  Block b;
  int part, parts;  // of the block's keys
  int slot;         // of the first part's results: those of a block follow each other
  int seam;         // divided blocks before this one
  int seams;        // divided blocks of all
};

// Part number `index`, of at most 256 sequences (SHARED); false: there are fewer.
template <int ROWS, int KEYS, bool PAGED>
__device__ __forceinline__ bool part_at(Args a, int index, int lane, Part& p) {
  constexpr int EACH = 4, UNDIVIDED = 1 << 26;
  int rows[EACH], keys[EACH], row0[EACH], key0[EACH], blocks[EACH], tiles[EACH];
#pragma unroll
  for (int e = 0; e < EACH; e++) {
    row0[e] = rows[e] = key0[e] = keys[e] = 0;
    if (64 * e < a.sequences && 64 * e + lane < a.sequences) {
      const Sequence q = sequence_at(a, 64 * e + lane, PAGED);
      row0[e] = q.row0, rows[e] = q.rows, key0[e] = q.key0, keys[e] = q.keys;
    }
    blocks[e] = (int)(((int64_t)rows[e] * a.group + ROWS - 1) / ROWS);
    tiles[e] = (keys[e] + KEYS - 1) / KEYS;
  }
  auto all_lanes = [&](int v) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(add_scan(v), 63); };
  // (parts of a block at C tiles to each: exact, as a list row's row is)
  auto parts_of = [&](int tiles, double inv, int most) __attribute__((always_inline)) {
    return max(1, (int)(((double)(tiles + most - 1) + 0.5) * inv));
  };
  int work = 0;
#pragma unroll
  for (int e = 0; e < EACH; e++) work += blocks[e] * min(tiles[e], 1 << 20);  // (blocks: fewer than 2^10)
  work = all_lanes(work);
  int most = max(a.least, (work + a.parts - 1) / a.parts);
  double inv = 0.0;
  for (int tries = 0;; tries++) {
    inv = 1.0 / (double)most;
    int n = 0, fewer = UNDIVIDED;  // the least that some block has a part less with
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int each = min(parts_of(tiles[e], inv, most), a.parts + 1);  // (so that the sum stays within 32 bits)
      n += blocks[e] * each;
      if (blocks[e] > 0 && each > 1) fewer = min(fewer, (int)((float)tiles[e] * __builtin_amdgcn_rcpf((float)(each - 1))) + 1);
    }
    n = all_lanes(n);
    if (n <= a.parts || most >= UNDIVIDED) break;
    // (larger in proportion, and so through in a few tries; where there are too many blocks nothing is divided in the end)
    most = tries < 8 ? max(max(most + 1, min_of_all(fewer)), uniform((int)fmin((double)most * n / a.parts, (double)UNDIVIDED)))
                     : UNDIVIDED;
  }
  int at = -1, before = 0, slots = 0, seams = 0;
#pragma unroll
  for (int e = 0; e < EACH; e++)
    if (64 * e < a.sequences) {
      const int each = parts_of(tiles[e], inv, most), mine = blocks[e] * each, divided = each > 1 ? blocks[e] : 0;
      const int upto = before + add_scan(mine), slots_upto = add_scan(divided * each), seams_upto = add_scan(divided);
      const uint64_t behind = __ballot(upto > index);
      if (at < 0 && behind) {
        at = __builtin_ctzll(behind);
        const int n = __builtin_amdgcn_readlane(blocks[e], at), parts = __builtin_amdgcn_readlane(each, at);
        const int in = index - (__builtin_amdgcn_readlane(upto, at) - n * parts), i = uniform(in / parts);
        p.b.q = {64 * e + at, __builtin_amdgcn_readlane(row0[e], at), __builtin_amdgcn_readlane(rows[e], at),
                 __builtin_amdgcn_readlane(key0[e], at), __builtin_amdgcn_readlane(keys[e], at)};
        // (the last blocks first: under the mask they have the most keys)
        p.b.block = n - 1 - i;
        p.parts = parts;
        p.part = in - i * parts;
        p.slot = slots + __builtin_amdgcn_readlane(slots_upto - divided * each, at) + (parts > 1 ? i * parts : 0);
        p.seam = seams + __builtin_amdgcn_readlane(seams_upto - divided, at) + (parts > 1 ? i : 0);
      }
      before = __builtin_amdgcn_readlane(upto, 63);
      slots += __builtin_amdgcn_readlane(slots_upto, 63);
      seams += __builtin_amdgcn_readlane(seams_upto, 63);
    }
  p.seams = seams;
  return at >= 0;
}

// One past the last key that some row of the block sees, and of one row.
__device__ __forceinline__ int end_of_row(Args a, const Sequence& q, int j) {
  return a.mask == ADR_MASK_CAUSAL ? clamp_to(j + q.keys - q.rows + 1, q.keys) : q.keys;
}


// A value that is no number times the zero of a key that a row does not see is no zero, and a page that is not in the cache is
// noticed for a block as a whole.  So where rows of a block come out as no numbers, the first of them seeing the keys before
// x0, this looks, by all lanes, whether some key of x0 ... x1 - 1, the block's last, holds such a value or has no page: then the rows
// are computed again from the keys that they see.  Otherwise it is their own result.  (For whole chunks of 16 bytes.)  One row
// after the other is slow, and these are a block's: a prompt of 4096 rows (32 / 8 heads of 128, 0.17 ms) whose first value is NaN
// 0.2 ms, whose 2000th or last one is 31 or 75 ms; with all rows that are no numbers computed again each took 75 to 89 ms.
__device__ __forceinline__ bool hidden_reaches(Args a, const Sequence& q, int hk, int x0, int x1, int lane) {
  const half_t* const V = a.v + hk * a.sv.z;
  bool lost = false;
  float zero = 0.0f;
  for (int x = x0 + lane; x < x1; x += 64) {
    int64_t ko, vo;
    if (!key_at(a, q, x, ko, vo)) {
      lost = true;
      break;
    }
    for (int i = 0; i < a.d; i += 8) {
      const half8_t v = *(const half8_t*)(V + vo + i);
#pragma unroll
      for (int e = 0; e < 8; e++) zero = fmaf((float)v[e], 0.0f, zero);
    }
  }
  return __ballot(lost || !(zero == 0.0f)) != 0;
}

// A transfer's descriptor, in scalar registers: `bytes` from an address on.
__device__ __forceinline__ u32x4_t descriptor(uint64_t p, int bytes) {
  return u32x4_t{(uint32_t)uniform((int)(uint32_t)p), (uint32_t)uniform((int)((uint32_t)(p >> 32) & 0xffffu)),
                 (uint32_t)uniform(bytes), 0x00020000u};
}

// One past the last key that all rows from row j on see, whatever their masks say.
__device__ __forceinline__ int end_of_common(Args a, const Sequence& q, int j) {
  return a.mask == MASK_TREE ? clamp_to(q.keys - q.rows, q.keys) : end_of_row(a, q, j);
}

// Sums the parts of the blocks that lie in several workgroups' stretches, in order: a workgroup to a seam, a thread to 4
// columns of a row, as many rows at once as 256 threads have.
template <int HD, int ROWS, bool U8 = false>
__global__ __launch_bounds__(256) void attention_join_kernel(Job) {
  constexpr int COLS = HD / 4, AT_ONCE = 256 / COLS < ROWS ? 256 / COLS : ROWS, GROUPS = ROWS / AT_ONCE;
  __shared__ int bad_rows;  // whose result is not finite; 16 bits on, whose scores are beyond FAR_SCORE
  static_assert(AT_ONCE <= 16, "a bit to each");
  const int tid = threadIdx.x, lane = tid & 63;
  Args a = arguments();
  const int hk = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  // (few rows: stretch s begins in slot 2 s, and the part before the seam is in front of that or of the one before)
  constexpr bool STRETCHES = ROWS == FEW;
  const int seam = rest / GROUPS + STRETCHES;
  const Seam b = a.seams[seam * a.kv_heads + hk];
  const int parts = b.parts, slot = b.slot, next = STRETCHES ? 2 * (seam - 1) : slot, step = STRETCHES ? 2 : 1;
  if (parts == 0) return;
  const int rows = min(ROWS, b.q.rows * a.group - b.block * ROWS), r0 = rest % GROUPS * AT_ONCE;
  if (r0 >= rows) return;
  // Few rows leave threads over: these share the parts.
  const int items = min(rows - r0, AT_ONCE) * COLS, sharers = 256 / items, sharer = tid / items, item = tid - sharer * items;
  const int r = r0 + item / COLS, col = item % COLS * 4;
  __shared__ float4_t sums[256];
  __shared__ float2 mls[256];
  if (tid == 0) bad_rows = 0;
  auto row_of = [&](int part) __attribute__((always_inline)) {
    return ((int64_t)(part == 0 ? slot : next + step * part) * a.kv_heads + hk) * ROWS + r;
  };
  float m = NO_SCORE, l = 0.0f;
  float4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
  if (sharer < sharers) {
    constexpr int UNROLL = 8;
    for (int s = sharer; s < parts; s += UNROLL * sharers) {
      float2 ml[UNROLL];
      float4_t v[UNROLL];
#pragma unroll
      for (int j = 0; j < UNROLL; j++) {
        const int64_t row = row_of(min(s + j * sharers, parts - 1));
        ml[j] = a.part_ml[row];
        v[j] = *(const float4_t*)(a.part_o + row * HD + col);
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < UNROLL; j++) top = fmaxf(top, ml[j].x);  // (the last part may be among them several times)
      const float alpha = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= alpha;
      acc *= alpha;
#pragma unroll
      for (int j = 0; j < UNROLL; j++)
        if (s + j * sharers < parts) {
          const float f = __builtin_amdgcn_exp2f(ml[j].x - m);
          l += ml[j].y * f;
          acc += v[j] * f;
        }
    }
  }
  sums[tid] = acc;
  mls[tid] = make_float2(m, l);
  __syncthreads();
  if (sharer == 0) {
    for (int s = 1; s < sharers; s++) {
      const float2 ml = mls[s * items + item];
      const float top = fmaxf(m, ml.x), f0 = __builtin_amdgcn_exp2f(m - top), f1 = __builtin_amdgcn_exp2f(ml.x - top);
      m = top;
      l = l * f0 + ml.y * f1;
      acc = acc * f0 + sums[s * items + item] * f1;
    }
    const int lr = b.block * ROWS + r, token = row_of_list(a, lr), h = hk * a.group + lr - token * a.group;
    half4_t out;
    const bool finite = round_means(out, acc, l == 0.0f ? 0.0f : 1.0f / l);
    if (!finite) atomicOr(&bad_rows, 1 << (r - r0));
    if (is_far(m)) atomicOr(&bad_rows, 0x10000 << (r - r0));
    if (col < a.d) *(half4_t*)(a.out + (int64_t)h * a.so_z + (int64_t)(b.q.row0 + token) * a.so_y + col) = out;
  }
  __syncthreads();
  int again = uniform(bad_rows) >> 16 & 0xffff;
  const int bad = uniform(bad_rows) & 0xffff;
  if (!U8 && bad && ((b.q.rows > 1 && a.mask == ADR_MASK_CAUSAL) || a.mask == MASK_TREE) &&
      hidden_reaches(a, b.q, hk, end_of_common(a, b.q, row_of_list(a, b.block * ROWS + r0 + __builtin_ctz(bad))),
                     end_of_row(a, b.q, row_of_list(a, b.block * ROWS + rows - 1)), lane))
    again |= bad;
  for (int x = tid >> 6; x < AT_ONCE; x += 4)
    if (again >> x & 1) {
      const int lr = b.block * ROWS + r0 + x;
      if constexpr (U8) row_by_wave_u8(arguments(), b.q, lr / a.group, hk * a.group + lr % a.group, lane);
      else row_by_wave(arguments(), b.q, lr / a.group, hk * a.group + lr % a.group, lane);
    }
}

}  // namespace
}  // namespace adr
