// Attention of packed rows of several sequences, over the pages of a cache or over packed keys.
//
//   out[h, row] = sum_x softmax_x( scale <q[h, row], k[x]> / temp ) v[x],   x <= j + n - r under the mask
//
// for row j of a sequence of r rows and n keys.  Query heads come in groups that share a key and value head.
#include <math.h>

#include <algorithm>
#include <type_traits>

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

// One row of one query head by one wavefront, at any strides: 64 keys at a time, a lane to a key for the scores
// and a lane to every 64th column for the sums.  Only keys that the row sees are read.  Probabilities stay in 32 bits, and
// scores unscaled until their maximum is subtracted: right for scores of any size.  (Columns col0 ... col1 - 1 are stored.)
constexpr int GENERAL_MAX_D = 256;
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
    if (x < end) {
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
    const int n = min(64, end - x0);
    for (int e = 0; e < n; e++) {
      const float pe = __shfl(p, e);
      const int64_t at = __shfl(vo, e);
      if (!__shfl((int)good, e)) {
#pragma unroll
        for (int c = 0; c < GENERAL_MAX_D / 64; c++) o[c] = NAN;
        continue;
      }
#pragma unroll
      for (int c = 0; c < GENERAL_MAX_D / 64; c++)
        if (c * 64 + lane < a.d) o[c] = fmaf(pe, (float)V[at + (c * 64 + lane) * a.sv.x], o[c]);
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
__global__ __launch_bounds__(256) void attention_any_layout_kernel(Job) {
  Args a = arguments();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i = (int64_t)blockIdx.x * 4 + wave; i < (int64_t)a.rows * a.heads; i += (int64_t)gridDim.x * 4) {
    const int h = (int)(i / a.rows), row = (int)(i - (int64_t)h * a.rows);
    const Sequence q = sequence_at(a, sequence_of_row(a.row_offsets, a.sequences, row, lane), a.table != nullptr);
    if (row < q.row0 || row >= q.row0 + q.rows) continue;
    row_by_wave(a, q, row - q.row0, h, lane);
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
template <int ROWS, int KEYS, bool PAGED, bool SHARED>
struct Roster {
  static constexpr int EACH = 4;
  typedef int each_t __attribute__((ext_vector_type(EACH)));
  each_t row0, rows, key0, keys;
  each_t upto;            // where on the line the sequence ends
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
        b.q = {base + 64 * e + at, __builtin_amdgcn_readlane(row0[e], at), __builtin_amdgcn_readlane(rows[e], at),
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

// ---- few rows: generation, a few tokens at once ----------------------------------------------------------
//
// A block of 16 rows against its keys: a read of the keys and values.  The workgroup's wavefronts walk tiles of
// 32 keys in turn, each through two tiles' worth of LDS of its own, so that the loop has no barrier.  S^T = K Q^T, so
// that a lane holds scores of one row, and O^T = V^T P^T, on MFMA 16x16x32; probabilities are rounded to fp16, the
// matrix cores' operands, sums and scores stay in 32 bits.  (fp16 probabilities cost 2^-11 of each; a product in 32 bits would be
// no matrix product, and its values are fp16 anyway.)
//
// Bound by memory: 16 rows of every key read once leave the matrix cores 5 % busy.  64 sequences of 3 to 4000 keys (32 / 8
// heads of 128, 504 MB) 88.2 us = 5.7 TB/s, eight of 50000 to 110000 (40 / 8, 2.36 GB) 365 us = 6.4 TB/s, where a plain read
// reaches 7.0 to 7.3; one of 777 keys (32 / 32) 9.6 to 10.4 us, of which two launches are 8.8 on the host.
template <int HD, bool PAGED, int WAVES, bool SHARED>
__global__ __launch_bounds__(64 * WAVES, 2) void attention_few_rows_kernel(Job) {
  constexpr int CPR = HD / 8, KEYS = 32, ROWS = 16;
  constexpr int ROWB = HD * 2, TILE = KEYS * ROWB;  // bytes of a tile row, of a K or V tile
  constexpr int NI = TILE / 1024;                   // transfers per tile
  constexpr int KS = HD / 32, DB = HD / 16;         // k-steps of S, blocks of 16 output columns
  constexpr int WAVE = 4 * TILE;                    // K0 K1 V0 V1 of a wavefront
  constexpr int PITCH = HD + 4;                     // of the partial results' rows, in floats
  constexpr int BIAS = NI / 2 * 1024;               // bytes that descriptors start ahead, so that no offset is negative
  static_assert(16 * (PITCH + 2) * 4 + 16 <= WAVE, "the partial results fit the tiles' LDS");
  // (WAVES * WAVE bytes, asked for at the launch: told of them, the compiler would count one wavefront to a SIMD, hand it
  // the accumulation registers as well and move every sum in and out of those)
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];

  Args first = arguments();
  early<PAGED, !SHARED>(first);
  const int kv_heads = first.kv_heads, hk = blockIdx.x % kv_heads, wg = blockIdx.x / kv_heads;
  Roster<ROWS, KEYS, PAGED, SHARED> roster;
  const Line line = roster.line_of(first, threadIdx.x & 63);
  if (wg >= line.parts) {
    if (SHARED && threadIdx.x == 0) arguments().seams[wg * kv_heads + hk].parts = 0;
    return;
  }
  const int stretch0 = SHARED ? line.at(wg) : wg, stretch1 = SHARED ? line.at(wg + 1) : wg + 1;
  for (int place = stretch0, next_place;; place = next_place) {
  Args a = SHARED ? arguments() : first;
  const int tid = thread_index(), lane = tid & 63, w = uniform(tid >> 6);
  const int frow = lane & 15, g = lane >> 4;
  Block b;
  if (!roster.block_at(a, a.shift, place, lane, b)) {
    if (SHARED && place == stretch0 && tid == 0) a.seams[wg * kv_heads + hk].parts = 0;
    return;
  }
  if constexpr (SHARED)  // (by one wait, as above)
    asm volatile("" ::"s"(a.seams), "s"(a.group), "s"(a.per_head), "s"(a.mask), "s"(a.d), "s"(a.q), "s"(a.sq_y), "s"(a.sq_z),
                 "s"(a.k), "s"(a.v), "s"(a.sk.y), "s"(a.sk.z), "s"(a.sv.y), "s"(a.sv.z));
  const Sequence q = b.q;
  const int block = b.block, pieces = min(stretch1 - place, b.pieces - b.offset);
  const bool whole = pieces == b.pieces;
  next_place = place + pieces;
  if (SHARED && place == stretch0 && tid == 0) a.seams[wg * kv_heads + hk] = seam_at(line, wg, place, b);
  const int rows = min(ROWS, q.rows * a.group - block * ROWS);          // of the block
  const int list_row = block * ROWS + min(frow, rows - 1), row = row_of_list(a, list_row), gh = list_row - row * a.group;

  const int last_end = uniform(end_of_row(a, q, row_of_list(a, block * ROWS + rows - 1)));  // of the block's last row
  const int all = (last_end + KEYS - 1) / KEYS;
  const int tile0 = whole ? 0 : min(all, b.offset << line.shift);
  const int tile1 = b.offset + pieces == b.pieces ? all : min(all, (b.offset + pieces) << line.shift);
  const int row_end = min(last_end, tile1 * KEYS);
  const int tiles = max(0, (tile1 - tile0 - w + WAVES - 1) / WAVES);  // of this wavefront: tile0 + w + WAVES i

  const half_t* const K = a.k + hk * a.sk.z + (PAGED ? 0 : q.key0 * a.sk.y);
  const half_t* const V = a.v + hk * a.sv.z + (PAGED ? 0 : q.key0 * a.sv.y);
  const uint32_t lds0 = (uint32_t)(uintptr_t)ADR_LDS_PTR(smem) + w * WAVE;
  const unsigned char* const sm = smem + w * WAVE;
  // The queries' fragments, by way of the second tile of values, which comes after them: nothing waits for them before the
  // first keys are on their way.  (Chunks behind the head dimension are zeros below.)
  const int d = a.d, k_stride = (int)a.sk.y, v_stride = (int)a.sv.y;
  const half_t* const qrow =
      a.q + (int64_t)(hk * a.group + gh) * a.sq_z + (int64_t)(q.row0 + row) * a.sq_y;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    const int col = ks * 32 + g * 8;
    dma_global(lds0 + 3 * TILE + ks * 1024, qrow + (col < d ? col : 0));
  }
  // Byte offsets of a lane's chunks in 16 rows (the second 16 rows of a tile repeat them); chunks behind the head
  // dimension lie behind every descriptor's end and come as zeros.
  uint32_t koff[NI / 2], voff[NI / 2];
#pragma unroll
  for (int j = 0; j < NI / 2; j++) {
    int krow, kc;
    k_chunk_inv<CPR>(j * 64 + lane, krow, kc);
    const int vrow = (j * 64 + lane) / CPR, vc = (lane % CPR) ^ v_swz8<CPR>(vrow);
    const uint32_t ko = (uint32_t)((krow * k_stride + kc * 8) * 2 + BIAS - j * 1024);
    const uint32_t vo = (uint32_t)((vrow * v_stride + vc * 8) * 2 + BIAS - j * 1024);
    koff[j] = kc * 8 < d ? ko : 0x7fff0000u;
    voff[j] = vc * 8 < d ? vo : 0x7fff0000u;
  }
  // Where the keys and values of 32 of the wavefront's tiles lie, a lane to each 16 keys: their addresses are worked
  // out by the vector ALU once, not by scalar instructions for each tile.  (Addresses are even: an odd one says that there
  // are keys.)
  uint64_t k_at = 0, v_at = 0;
  bool lost = false;  // a key's page is not in the cache
  auto look_up = [&](int i) __attribute__((always_inline)) {
    const int key = (tile0 + w + WAVES * (i + (lane >> 1))) * KEYS + 16 * (lane & 1);
    k_at = v_at = 0;  // (no keys)
    if (key < row_end) {
      int64_t ko = key * a.sk.y, vo = key * a.sv.y;
      bool good = true;
      if constexpr (PAGED) {
        const int page = a.table[(int64_t)q.index * a.table_pitch + (key >> a.page_shift)];
        const int slot = key & ((1 << a.page_shift) - 1);
        good = page >= 0 && page < a.pages;
        ko = page * a.sk.p + slot * a.sk.y;
        vo = page * a.sv.p + slot * a.sv.y;
      }
      lost |= !good;
      if (good) k_at = ((uint64_t)(K + ko) - BIAS) | 1, v_at = ((uint64_t)(V + vo) - BIAS) | 1;
    }
  };
  // Keys, or values, of tile i.
  auto fetch = [&](int i, auto is_k) __attribute__((always_inline)) {
    constexpr bool IS_K = decltype(is_k)::value;
    const int stride = IS_K ? k_stride : v_stride;
    const uint64_t at = IS_K ? k_at : v_at;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int l = 2 * (i & 31) + h, left = min(row_end - (tile0 + w + WAVES * i) * KEYS - 16 * h, 16);
      const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at, l), hi = __builtin_amdgcn_readlane((uint32_t)(at >> 32), l);
      const u32x4_t desc = {lo & ~1u, hi & 0xffffu, lo & 1 ? (uint32_t)(((left - 1) * stride + d) * 2 + BIAS) : 0u, 0x00020000u};
      dma_buffer_once<NI / 2>(lds0 + ((IS_K ? 0 : 2) + (i & 1)) * TILE + h * (NI / 2) * 1024, IS_K ? koff : voff, desc);
    }
  };
  const std::true_type is_k{};
  const std::false_type is_v{};

  look_up(0);
  // (the lookup's load has landed before the transfers' own count begins)
  if (tiles > 0) fetch(0, is_k), fetch(0, is_v);
  if (tiles > 1) fetch(1, is_k);
  if (tiles > 1) wait_vm<3 * NI>();
  else if (tiles > 0) wait_vm<2 * NI>();
  else wait_vm<0>();
  half8_t qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    qf[ks] = *(const half8_t*)(sm + 3 * TILE + ks * 1024 + lane * 16);
    if (ks * 32 + g * 8 >= d) qf[ks] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(qf[ks]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (tiles > 1) fetch(1, is_v);
  int offK[KS], offV[DB];
#pragma unroll
  for (int ks = 0; ks < KS; ks++) offK[ks] = k_chunk_off<CPR>(frow, ks * 4 + g);
  {
    const int c = lane & 15, r = 4 * g + (c >> 2);
#pragma unroll
    for (int db = 0; db < DB; db++)
      offV[db] = r * ROWB + (((2 * db + ((c & 3) >> 1)) ^ v_swz8<CPR>(r)) << 4) + (c & 1) * 8;
  }
  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4_t;

  float4_t o[DB];
  float m_run = NO_SCORE, l_run = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; db++) o[db] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int end = min(end_of_row(a, q, row), row_end) - 4 * g;  // this lane's first key that its row does not see
  // Tile i; `next`: there is a tile i + 1, `more`: and a tile i + 2, whose keys and values are asked for as soon as the
  // fragments of this one's are in registers.
  auto tile = [&](int i, auto next, auto more) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value, MORE = decltype(more)::value;
    wait_vm<NEXT ? 3 * NI : NI>();  // its keys have landed
    const unsigned char* const cK = sm + (i & 1) * TILE;
    const unsigned char* const cV = sm + (2 + (i & 1)) * TILE;
    float4_t s[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int kb = 0; kb < 2; kb++) {
        const half8_t kf = *(const half8_t*)(cK + offK[ks] + kb * 16 * ROWB);
        s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[ks], s[kb], 0, 0, 0);
      }
    if constexpr (MORE) {
      if (((i + 2) & 31) == 0) look_up(i + 2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fetch(i + 2, is_k);
    }
    wait_vm<MORE ? 3 * NI : NEXT ? 2 * NI : 0>();  // and its values
    half8_t vf[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) {
      const unsigned char* const p0 = cV + offV[db];
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0 + 16 * ROWB));
      vf[db] = __builtin_shufflevector(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, hi),
                                       0, 1, 2, 3, 4, 5, 6, 7);
    }
    if constexpr (MORE) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int db = 0; db < DB; db++) asm volatile("" : "+v"(vf[db]));
      fetch(i + 2, is_v);
    }
    const int left = end - (tile0 + w + WAVES * i) * KEYS;  // keys of this lane's row from its first one on
    float mx = NO_SCORE;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        if (16 * kb + r >= left) s[kb][r] = -INFINITY;
        mx = fmaxf(mx, s[kb][r]);
      }
    float x = mx, y = mx;  // over the four lanes that share a row
    swap_halves(x, y);
    x = fmaxf(x, y), y = x;
    swap_rows(x, y);
    const float top = above(fmaxf(x, y) * a.c);
    if (__builtin_amdgcn_ballot_w64(top > m_run + GROWN) != 0) {
      const float m_new = fmaxf(m_run, top - BELOW), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; db++) o[db] *= alpha;
    }
    float sum[2] = {0.0f, 0.0f};
    u32x4_t pf;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float2_t e;
#pragma unroll
        for (int j = 0; j < 2; j++) {
          e[j] = __builtin_amdgcn_exp2f(fmaf(s[kb][r + j], a.c, -m_run));
          sum[j] += e[j];
        }
        pf[kb * 2 + r / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(e, half2_t));
      }
    l_run += sum[0] + sum[1];
#pragma unroll
    for (int db = 0; db < DB; db++)
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[db], __builtin_bit_cast(half8_t, pf), o[db], 0, 0, 0);
  };
  const std::true_type yes{};
  const std::false_type no{};
  int i = 0;
  for (; i + 2 < tiles; i++) tile(i, yes, yes);
  if (i + 1 < tiles) tile(i++, yes, no);
  if (i < tiles) tile(i, no, no);

  Args z = arguments();
  // Merge the wavefronts' results: [wavefront][row][HD] sums, and (maximum, sum) of every row.
  wait_vm<0>();
  __syncthreads();
  float* const xo = (float*)smem;
  float2* const xml = (float2*)(smem + WAVES * 16 * PITCH * 4);
  int* const bad_rows = (int*)(smem + WAVES * 16 * (PITCH + 2) * 4);  // rows whose result is not finite
  float x = l_run, y = x;
  swap_halves(x, y);
  x = x + y, y = x;
  swap_rows(x, y);
  if (__ballot(lost)) x = NAN;
  if (tid == 0) *bad_rows = 0;
  if (g == 0) xml[w * 16 + frow] = make_float2(m_run, x + y);
#pragma unroll
  for (int db = 0; db < DB; db++) *(float4_t*)(xo + (w * 16 + frow) * PITCH + 16 * db + 4 * g) = o[db];
  __syncthreads();
  for (int e = tid; e < rows * (HD / 4); e += 64 * WAVES) {
    const int r = e / (HD / 4), col = e % (HD / 4) * 4;
    float2 ml[WAVES];
    float m_all = NO_SCORE, l = 0.0f;
#pragma unroll
    for (int x = 0; x < WAVES; x++) {
      ml[x] = xml[x * 16 + r];
      m_all = fmaxf(m_all, ml[x].x);
    }
    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < WAVES; x++) {
      const float f = __builtin_amdgcn_exp2f(ml[x].x - m_all);
      l += ml[x].y * f;
      sum += *(const float4_t*)(xo + (x * 16 + r) * PITCH + col) * f;
    }
    if (whole) {
      const int lr = block * ROWS + r, token = row_of_list(z, lr), h = hk * z.group + lr - token * z.group;
      half4_t v;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (!round_means(v, sum, inv)) atomicOr(bad_rows, 1 << r);
      if (col < z.d && !is_far(m_all))
        *(half4_t*)(z.out + (int64_t)h * z.so_z + (int64_t)(q.row0 + token) * z.so_y + col) = v;
    } else {
      const int64_t prow = ((int64_t)(2 * wg + (place != stretch0)) * z.kv_heads + hk) * ROWS + r;
      *(float4_t*)(z.part_o + prow * HD + col) = sum;
      if (col == 0) z.part_ml[prow] = make_float2(m_all, l);
    }
  }
  if (whole) {
    float m_all = NO_SCORE;
#pragma unroll
    for (int x = 0; x < WAVES; x++) m_all = fmaxf(m_all, xml[x * 16 + frow].x);
    int again = (int)__ballot(is_far(m_all));  // (not stored above)
    if (q.rows > 1 && z.mask == ADR_MASK_CAUSAL) {
      __syncthreads();
      const int bad = uniform(*bad_rows);
      if (bad && hidden_reaches(z, q, hk, end_of_row(z, q, row_of_list(z, block * ROWS + __builtin_ctz(bad))),
                                end_of_row(z, q, row_of_list(z, block * ROWS + rows - 1)), lane))
        again |= bad;
    }
    for (int r = w; r < rows; r += WAVES)
      if (again >> r & 1) {
        const int lr = block * ROWS + r;
        row_by_wave(arguments(), q, lr / z.group, hk * z.group + lr % z.group, lane);
      }
  }
  if (!SHARED || next_place >= stretch1) break;
  __syncthreads();  // (the next block's transfers go where the results are read)
  }
}

// ---- many rows: prompts, and their pieces over what is in the cache ---------------------------------------
//
// A workgroup takes a block of 128 rows, wavefront w of it rows 32 w ... 32 w + 31 of the list, and walks tiles of 64
// keys, double buffered in LDS by transfers from global memory; two workgroups share a compute unit.  Per tile a
// wavefront computes S^T = K Q^T (MFMA 32x32x16, Q fragments resident in registers), so that every lane holds scores
// of one row: the running maximum and sum are in-lane reductions plus one exchange with lane ^ 32, and a lane's own
// last key is all that the mask needs.  The probabilities, narrowed to fp16, are already in the operand layout of the
// second product O^T = V^T P^T, whose V^T fragments come from the row-major V tile by transposing LDS reads.  The two
// products and the softmax between them are one instruction stream, as in attention_fwd_kernel (attention.hip, which
// explains the arrangement): scores of tile i + 1 on the matrix cores beside the exponentials of tile i, P.V of tile i
// beside the maximum of tile i + 1.  What is different here is where rows and keys come from: the heads of a group
// share the block, so that a key row is read once for all of them and the part of a tile that the mask leaves empty
// is 1 / group as wide, and each wavefront's 16 key rows of a tile have a base address of their own, on a page.
//
// GROUPS == 2: eight wavefronts, of which four take the first half of the block's keys and four the second, each through
// tiles of its own; both ends meet in LDS.  Two workgroups beside each other do as much, but that takes twice as many blocks,
// or parts that go through memory: 1024 rows over 8025 keys (256 blocks) 134 us, by halves through memory 143, one group on
// each compute unit 144 (all three on one machine).
//
// Bound by issue as in attention_fwd_kernel, and where all is loop by power: one prompt of 16384 rows (32 / 8 heads of 128) 2006
// to 2196 us by machine = 1096 to 1000 TFLOP/s, with the matrix cores busy 69 % of cycles at 1.6 GHz, where a product of 8192^3
// reaches 1408.  The 256 blocks above, two groups each, leave some of that power: 53 % at 1.8 GHz, 136 to 146 us.  Short blocks are
// bound by their beginnings and ends: us of a block among others, 2.0 from the end of one to the start of the next in its place,
// 1.4 to find its sequence, 1.7 for addresses, 1.8 until the first keys are there, 1.9 a tile, 2.4 for the results.  Nine prompts
// of 100 to 3996 rows, 25 tiles a block in the mean, 447 to 477 us = 933 to 874 TFLOP/s (what wavefronts whose rows end early, and
// rows that the mask hides, compute of a tile is in the time and not in the operations).  HD = 128 keeps 24 to 38 vector registers
// in scratch memory at those beginnings and ends, none in the loop; HD = 64 none.
template <int HD, bool PAGED, bool SHARED, int GROUPS>
__global__ __launch_bounds__(256 * GROUPS, 2) void attention_tiles_kernel(Job) {
  constexpr int CPR = HD / 8, KEYS = 64, ROWS = 128;
  constexpr int TILE = KEYS * HD * 2;  // bytes of one K or V tile
  constexpr int NI = TILE / 1024 / 4;  // transfers per wavefront and tile: 16 rows
  constexpr int DS = HD / 16;          // MFMA k-steps over the head dimension
  constexpr int DT = HD / 32;          // 32-wide output column tiles
  constexpr int ROWB = HD * 2;         // bytes per tile row
  constexpr int BIAS = NI * 1024;      // bytes that descriptors start ahead, so that no offset is negative
  __shared__ __attribute__((aligned(1024))) unsigned char smem[GROUPS * 4 * TILE];  // K0 K1 V0 V1 of each group
  __shared__ int lost_keys[4 * GROUPS];  // of each wavefront

  // Consecutive workgroups go to different dies; where the key heads divide evenly, a die takes its share of them, so
  // that the blocks which read the same keys meet in one L2.
  Args a = arguments();
  early<PAGED>(a);
  const int kv_heads = a.kv_heads;
  int hk, index;
  if (kv_heads % 8 == 0) {
    const int each = kv_heads >> 3, seq = blockIdx.x >> 3;
    hk = (blockIdx.x & 7) * each + seq % each;
    index = seq / each;
  } else {
    hk = blockIdx.x % kv_heads;
    index = blockIdx.x / kv_heads;
  }
  const int tid = threadIdx.x, lane = tid & 63, group = GROUPS == 1 ? 0 : uniform(tid >> 8), w = uniform(tid >> 6 & 3);
  const int frow = lane & 31, g = lane >> 5;
  Part pt = {{}, 0, 1, 0, 0, 0};
  if constexpr (SHARED) {
    const bool some = part_at<ROWS, KEYS, PAGED>(a, index, lane, pt);
    // (the second launch has a workgroup to each two slots)
    if (tid == 0 && index >= pt.seams && index < a.parts / 2) a.seams[index * kv_heads + hk].parts = 0;
    if (!some) return;
    if (tid == 0 && pt.part == 0 && pt.parts > 1) a.seams[pt.seam * kv_heads + hk] = Seam{pt.parts, pt.slot, pt.b.q, pt.b.block};
  } else {
    Roster<ROWS, KEYS, PAGED, false> roster;
    roster.load(a, 0, lane, 0, 0);
    if (!roster.block_at(a, 0, index, lane, pt.b)) return;
  }
  const Sequence q = pt.b.q;
  const int block = pt.b.block, part = pt.part, parts = pt.parts, slot0 = pt.slot;
  const int rows = min(ROWS, q.rows * a.group - block * ROWS);  // of the block
  const int wave_rows = min(32, rows - w * 32);                 // of the wavefront (may be negative)
  const int list0 = block * ROWS + w * 32;
  // (lanes without a row of their own compute the block's last one)
  const int list_row = block * ROWS + min(w * 32 + frow, rows - 1), row = row_of_list(a, list_row), gh = list_row - row * a.group;
  const int lane_end = end_of_row(a, q, row);
  unsigned char* const sm = smem + group * (4 * TILE);
  const uint32_t lds0 = (uint32_t)(uintptr_t)ADR_LDS_PTR(smem) + group * (4 * TILE);
  const int d = a.d, k_stride = (int)a.sk.y, v_stride = (int)a.sv.y;
  // The queries' fragments, by way of the values' LDS, so that nothing waits for them before the first keys are on their
  // way.  (Chunks behind the head dimension are zeros below.)
  static_assert(4 * DS * 1024 <= 2 * TILE, "the queries fit the values' tiles");
  const half_t* const qrow = a.q + (int64_t)(hk * a.group + gh) * a.sq_z + (int64_t)(q.row0 + row) * a.sq_y;
#pragma unroll
  for (int ds = 0; ds < DS; ds++) {
    const int col = ds * 16 + g * 8;
    dma_global(lds0 + 2 * TILE + (w * DS + ds) * 1024, qrow + (col < d ? col : 0));
  }

  const int last_end = uniform(end_of_row(a, q, row_of_list(a, block * ROWS + rows - 1)));
  const int all = (last_end + KEYS - 1) / KEYS;
  // (exact, as above)
  auto cut = [&](int i) __attribute__((always_inline)) { return uniform((int)((double)all * (double)i / (double)parts)); };
  const int part0 = SHARED ? cut(part) : 0, part_tiles = (SHARED ? cut(part + 1) : all) - part0;
  // (of each group; the second may have one less)
  const int steps = (part_tiles + GROUPS - 1) / GROUPS, tile0 = part0 + group * steps;
  const int row_end = min(last_end, min(part0 + part_tiles, tile0 + steps) * KEYS);
  // Tiles that this wavefront computes: none without rows, none whose first key lies beyond its last row's.
  int active = 0, first_edge = 0;
  if (wave_rows > 0) {
    active = uniform(clamp_to((end_of_row(a, q, row_of_list(a, list0 + wave_rows - 1)) + KEYS - 1) / KEYS - tile0, min(steps, part0 + part_tiles - tile0)));
    // the first of them with keys that some row of the wavefront must not see
    first_edge = uniform(end_of_row(a, q, row_of_list(a, list0))) / KEYS - tile0;
  }

  // Wavefront w transfers rows 16 w ... 16 w + 15 of a tile, 1 KiB at a time: byte offsets of a lane's chunks in those
  // rows, less the j KiB that the instruction adds; chunks behind the head dimension come as zeros.
  uint32_t koff[NI], voff[NI];
#pragma unroll
  for (int j = 0; j < NI; j++) {
    int krow, kc;
    k_chunk_inv<CPR>(j * 64 + lane, krow, kc);
    const int vrow = (j * 64 + lane) / CPR, vc = (lane % CPR) ^ v_swz<CPR>(vrow);
    const uint32_t ko = (uint32_t)((krow * k_stride + kc * 8) * 2 + BIAS - j * 1024);
    const uint32_t vo = (uint32_t)((vrow * v_stride + vc * 8) * 2 + BIAS - j * 1024);
    koff[j] = kc * 8 < d ? ko : 0x7fff0000u;
    voff[j] = vc * 8 < d ? vo : 0x7fff0000u;
  }
  // The wavefront's next 16 key and value rows: address, and bytes from there to the last key (0 behind it).  On
  // pages, the addresses of 64 tiles at a time, a lane to each, worked out by the vector ALU.  (Addresses are even: an
  // odd one says that there is one.)  Keys are ahead of values: theirs bring the pages, which the values take over.
  struct Next {
    uint64_t base, p, pages;
    int64_t page_stride;
    int bytes, key, stride;
  };
  bool lost = false;  // a key's page is not in the cache
  int page = 0;
  auto locate = [&](Next& t, auto is_k) __attribute__((always_inline)) {
    const int left = min(row_end - t.key, 16);
    t.bytes = left > 0 ? ((left - 1) * t.stride + d) * 2 + BIAS : 0;
    if constexpr (PAGED) {
      const int n = ((t.key - 16 * w) >> 6) - tile0;
      if ((n & 63) == 0) {
        const int key = t.key + lane * KEYS;
        if constexpr (decltype(is_k)::value) {
          page = -1;
          if (key < row_end) {
            page = a.table[(int64_t)q.index * a.table_pitch + (key >> a.page_shift)];
            if (page < 0 || page >= a.pages) lost = true, page = -1;
          }
        }
        const int slot = key & ((1 << a.page_shift) - 1);
        t.pages = page < 0 ? 0 : (t.base + 2 * (page * t.page_stride + slot * (int64_t)t.stride)) | 1;
      }
      const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)t.pages, n & 63);
      const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(t.pages >> 32), n & 63);
      t.p = (uint64_t)hi << 32 | (lo & ~1u);
      if (!(lo & 1)) t.bytes = 0;
    }
  };
  const std::true_type is_k{};
  const std::false_type is_v{};
  auto first_tile = [&](const half_t* base, int64_t stride, int64_t page_stride, auto k) __attribute__((always_inline)) {
    Next t;
    t.base = (uint64_t)(base + (PAGED ? 0 : q.key0 * stride)) - BIAS;
    t.page_stride = page_stride;
    t.stride = (int)stride;
    t.key = tile0 * KEYS + 16 * w;
    t.pages = 0;
    t.p = t.base + 2 * (t.key * stride);
    locate(t, k);
    return t;
  };
  Next nk = first_tile(a.k + hk * a.sk.z, a.sk.y, a.sk.p, is_k), nv = first_tile(a.v + hk * a.sv.z, a.sv.y, a.sv.p, is_v);
  auto advance = [&](Next& t, auto k) __attribute__((always_inline)) {
    t.key += KEYS;
    if constexpr (!PAGED) t.p += (uint32_t)t.stride * (KEYS * 2u);
    locate(t, k);
  };
  // Transfers 2 j and 2 j + 1 of the NI that bring a tile into buffer `buf` (0, 1: K; 2, 3: V).
  auto transfer = [&](const Next& t, auto is_k, int buf, auto pair) __attribute__((always_inline)) {
    constexpr int J = 2 * decltype(pair)::value;
    const uint32_t dst = lds0 + w * (NI * 1024) + buf * TILE;
    const u32x4_t desc = descriptor(t.p, t.bytes);
    if constexpr (decltype(is_k)::value) dma_buffer_pair<J>(dst, koff[J], koff[J + 1], desc);
    else dma_buffer_pair<J>(dst, voff[J], voff[J + 1], desc);
  };
  const std::integral_constant<int, 0> pair0{};
  const std::integral_constant<int, NI / 2 - 1> pair1{};  // (the last pair; HD = 64 has one)
  auto tile_transfers = [&](Next& t, auto k, int buf) __attribute__((always_inline)) {
    transfer(t, k, buf, pair0);
    if constexpr (NI > 2) transfer(t, k, buf, pair1);
    advance(t, k);
  };
  // What is waited for at the end of each half: all transfers but those issued in it.
  auto wait_landed = [&]() __attribute__((always_inline)) { wait_vm<NI>(); };

  tile_transfers(nk, is_k, 0);
  tile_transfers(nk, is_k, 1);
  // LDS fragment offsets.  K: lane -> tile row frow (+32), chunk 2*ds + g.
  int offK[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ds++) offK[ds] = k_chunk_off<CPR>(frow, ds * 2 + g);
  wait_vm<NI>();  // the queries and the first K tile have landed
  half8_t qf[DS];  // (operand B of S^T = K Q^T: lane -> row frow, head-dimension group g)
#pragma unroll
  for (int ds = 0; ds < DS; ds++) {
    qf[ds] = *(const half8_t*)(sm + 2 * TILE + (w * DS + ds) * 1024 + lane * 16);
    if (ds * 16 + g * 8 >= d) qf[ds] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int ds = 0; ds < DS; ds++) asm volatile("" : "+v"(qf[ds]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (values come there behind the next barrier)
  // V (transposing read): in each group of 16 lanes, lanes 4r..4r+3 address 16 consecutive halves of tile row r, and
  // lane i of the group receives column i of that 4 x 16 block.  Group b = (lane / 16) % 2 takes columns 16b.. of the
  // 32-column tile, g the rows 4g..4g+3.
  int offV[DT];
  {
    const int s = lane & 15, b = (lane >> 4) & 1, r = s >> 2;
    const int row = 4 * g + r;  // + 32*kt + 16*t + 8*h, all multiples of 8: row & 3 == r
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      const int chunk = 4 * dt + 2 * b + ((s & 3) >> 1);
      offV[dt] = row * ROWB + ((chunk ^ v_swz<CPR>(row)) << 4) + (s & 1) * 8;
    }
  }

  float16_t o[DT], sa[2], sb[2];  // sums of P.V; scores of two tiles in turn
  u32x4_t pf[2][2];                 // probabilities, two to a register
#pragma unroll
  for (int dt = 0; dt < DT; dt++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[dt][r] = 0.0f;
  float m_run = NO_SCORE, l_run = 0.0f;  // running maximum (log2 units) and this lane's sum

  typedef short short4_t __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) short4_t lds_short4_t;
  // A half tile is NG groups of four MFMAs.  A group's fragments are read a group ahead, and used in
  // the opposite order, so that one wait covers all four.
  constexpr int NG = DS / 2;
  half8_t kf[NG][4], vf[NG][4];

  auto read_k = [&](const unsigned char* cK, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; j++) kf[c][j] = *(const half8_t*)(cK + offK[2 * c + (j >> 1)] + (j & 1) * 32 * ROWB);
  };
  // which of the products with V the j-th of group c is: keys 32 kt + 16 t ..., columns 32 dt ...
  auto pv_of = [](int c, int j, int& kt, int& t, int& dt) __attribute__((always_inline)) {
    const int p = 4 * c + j;
    kt = p / (2 * DT), t = p / DT % 2, dt = p % DT;
  };
  auto read_v = [&](const unsigned char* cV, int c) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; j++) {
      int kt, t, dt;
      pv_of(c, j, kt, t, dt);
      const unsigned char* p0 = cV + offV[dt] + (32 * kt + 16 * t) * ROWB;
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0 + 8 * ROWB));
      vf[c][j] = __builtin_shufflevector(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, hi),
                                         0, 1, 2, 3, 4, 5, 6, 7);
    }
  };

  // First half of tile i: the scores of tile i + 1 on the matrix cores (K buffer KB), and the
  // probabilities of tile i on the vector ALU.
  auto half1 = [&](auto do_s, auto do_p, auto do_pv, auto kbuf, float16_t (&cur)[2], float16_t (&nxt)[2])
                   __attribute__((always_inline)) {
    constexpr bool S = decltype(do_s)::value, P = decltype(do_p)::value;
    constexpr int KB = decltype(kbuf)::value, VB = 1 - KB;
    const unsigned char* const cK = sm + KB * TILE;
    const unsigned char* const cV = sm + (2 + VB) * TILE;
    // Piece k of the softmax: VP scores, in three stages that run a piece apart, so that no instruction
    // waits for the one before it: exponents (k + 1), powers of two (k), rounding and sum (k - 1).
    // (The empty assembly keeps the stages where they are.  Sums by v_dot2 would be half the
    // instructions, but those wait for the matrix cores.)
    constexpr int NP = 4 * NG, VP = 32 / NP;
    float sum[2] = {l_run, 0.0f};
    float ex[VP], pw[VP];
    auto stage_exponent = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e++) ex[e] = fmaf(cur[k * VP >> 4][(k * VP & 15) + e], a.c, -m_run);
    };
    auto stage_power = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e++) pw[e] = __builtin_amdgcn_exp2f(ex[e]);
    };
    auto stage_round = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e += 2) {
        const int x = k * VP + e;
        const float2_t e2 = {pw[e], pw[e + 1]};
        uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(e2, half2_t));
        sum[0] += pw[e];
        sum[1] += pw[e + 1];
        asm volatile("" : "+v"(bits), "+v"(sum[0]), "+v"(sum[1]));
        pf[x >> 4][x >> 3 & 1][(x & 7) / 2] = bits;
      }
    };
    if constexpr (HD == 128) __builtin_amdgcn_s_setprio(1);
    if constexpr (P) stage_exponent(0);
    if constexpr (S) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int r = 0; r < 16; r++) nxt[kt][r] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < NG; c++) {
      if constexpr (S) {
        if (c + 1 < NG) read_k(cK, c + 1);
      }
      if constexpr (decltype(do_pv)::value) {
        if (c + 1 == NG) read_v(cV, 0);
      }
      if (c == 0) transfer(nv, is_v, 2 + KB, pair0);
      if constexpr (NI > 2) {
        if (c == NG / 2) transfer(nv, is_v, 2 + KB, pair1);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (S) {
          constexpr int last = 3;
          const int f = last - j;
          nxt[f & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c][f], qf[2 * c + (f >> 1)], nxt[f & 1], 0, 0, 0);
        }
        if constexpr (P) {
          const int k = 4 * c + j;
          if (k > 0) stage_round(k - 1);
          stage_power();
          if (k + 1 < NP) stage_exponent(k + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (P) {
      stage_round(NP - 1);
      l_run = sum[0] + sum[1];
      asm volatile("" : "+v"(l_run));
    }
    if constexpr (HD == 128) __builtin_amdgcn_s_setprio(0);
    advance(nv, is_v);
    wait_landed();
    barrier();
  };

  // Second half of tile i: P.V of tile i on the matrix cores (V buffer VB), and the maximum of the
  // scores of tile i + 1 on the vector ALU.
  auto half2 = [&](int i, auto do_pv, auto do_max, auto do_s, auto vbuf, float16_t (&nxt)[2])
                   __attribute__((always_inline)) {
    constexpr bool PV = decltype(do_pv)::value, MAX = decltype(do_max)::value;
    constexpr int VB = decltype(vbuf)::value, KB = VB;  // K buffer of tile i + 2
    const unsigned char* const cV = sm + (2 + VB) * TILE;
    const unsigned char* const cK = sm + KB * TILE;
    if constexpr (MAX) {
      if (i + 1 >= first_edge) {
        // this lane's first masked key, counted from its own first one
        int end = lane_end - (tile0 + i + 1) * KEYS - 4 * g;
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            asm volatile("" : "+v"(end));  // (one comparison at a time: 32 would take as many scalar register pairs)
            if (32 * kt + 8 * (r >> 2) + (r & 3) >= end) nxt[kt][r] = -INFINITY;
          }
      }
    }
    // (the maximum from the second group on, when the scores are there; done before the last one)
    constexpr int FIRST = NG == 4 ? 4 : 2, PER = NG == 4 ? 2 : 4;
    float mx2[2] = {NO_SCORE, NO_SCORE}, mx = 0.0f;
#pragma unroll
    for (int c = 0; c < NG; c++) {
      if constexpr (PV) {
        if (c + 1 < NG) read_v(cV, c + 1);
      }
      if constexpr (decltype(do_s)::value) {
        if (c + 1 == NG) read_k(cK, 0);
      }
      if (c == 0) transfer(nk, is_k, 1 - KB, pair0);
      if constexpr (NI > 2) {
        if (c == NG / 2) transfer(nk, is_k, 1 - KB, pair1);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (PV) {
          constexpr int last = 3;
          const int f = last - j;
          int kt, t, dt;
          pv_of(c, f, kt, t, dt);
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[c][f], __builtin_bit_cast(half8_t, pf[kt][t]), o[dt], 0, 0, 0);
        }
        if constexpr (MAX) {
          const int first = (4 * c + j - FIRST) * PER * 2;
          if (first >= 0 && first < 32) {
#pragma unroll
            for (int e = 0; e < PER; e++) {
              const int x = first + 2 * e;
              mx2[e & 1] = fmaxf(fmaxf(mx2[e & 1], nxt[x >> 4][x & 15]), nxt[x >> 4][(x & 15) + 1]);
            }
          }
          if (first == 32) mx = above(pair_max(fmaxf(mx2[0], mx2[1])) * a.c);  // in log2 units (c > 0)
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (MAX) {
      if (__builtin_amdgcn_ballot_w64(mx > m_run + GROWN) != 0) {
        const float m_new = fmaxf(m_run, mx - BELOW);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[dt][r] *= alpha;
      }
    }
    advance(nk, is_k);
    wait_landed();
    barrier();
  };
  auto idle = [&](int i) __attribute__((always_inline)) {
    tile_transfers(nv, is_v, 2 + ((i + 1) & 1));
    wait_landed();
    barrier();
    tile_transfers(nk, is_k, (i + 1) & 1);
    wait_landed();
    barrier();
  };

  const std::true_type yes{};
  const std::false_type no{};
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};

  barrier();  // the first K tile has landed for every wavefront
  int i = -1;
  if (active > 0) {
    read_k(sm, 0);
    half1(yes, no, no, even, sb, sa);
    half2(-1, no, yes, yes, odd, sa);
    for (i = 0; i + 2 < active; i += 2) {
      half1(yes, yes, yes, odd, sa, sb);
      half2(i, yes, yes, yes, even, sb);
      half1(yes, yes, yes, even, sb, sa);
      half2(i + 1, yes, yes, yes, odd, sa);
    }
    if (i + 1 < active) {
      half1(yes, yes, yes, odd, sa, sb);
      half2(i, yes, yes, no, even, sb);
      half1(no, yes, yes, even, sb, sa);
      half2(i + 1, yes, no, no, odd, sa);
    } else {
      half1(no, yes, yes, odd, sa, sb);
      half2(i, yes, no, no, even, sb);
    }
    i = active;
  }
  for (; i < steps; i++) idle(i);  // tiles this wavefront has no part in
  wait_vm<0>();  // (transfers of no bytes write zeros)
  if constexpr (PAGED) {
    if (lane == 0) lost_keys[4 * group + w] = __ballot(lost) != 0;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  barrier();  // every read of K and V tiles is done: LDS is free

  // The groups' sums are joined by way of LDS: each finishes half of the columns.
  constexpr int MINE = DT / GROUPS;
  constexpr int EXCHANGE = GROUPS == 1 ? 0 : 256 * MINE * 64;  // bytes from a group
  float16_t res[MINE];
  if constexpr (GROUPS == 2) {
    __shared__ float2 mls[2][256];
    const int at = tid & 255;
    float4_t* const theirs = (float4_t*)(smem + (1 - group) * (4 * TILE)) + at;
    float4_t* const ours = (float4_t*)sm + at;
    auto give = [&](auto first) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < MINE; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float16_t& v = o[decltype(first)::value + d];
          ours[(4 * d + i) * 256] = float4_t{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        }
    };
    if (group == 0) give(std::integral_constant<int, MINE>{});
    else give(std::integral_constant<int, 0>{});
    mls[group][at] = make_float2(m_run, l_run);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    barrier();
    const float2 ml = mls[1 - group][at];
    const float top = fmaxf(m_run, ml.x), f0 = __builtin_amdgcn_exp2f(m_run - top), f1 = __builtin_amdgcn_exp2f(ml.x - top);
    m_run = top;
    l_run = l_run * f0 + ml.y * f1;
    auto take = [&](auto first) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < MINE; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float16_t& v = o[decltype(first)::value + d];
          const float4_t x = theirs[(4 * d + i) * 256];
#pragma unroll
          for (int j = 0; j < 4; j++) res[d][4 * i + j] = v[4 * i + j] * f0 + x[j] * f1;
        }
    };
    if (group == 0) take(std::integral_constant<int, 0>{});
    else take(std::integral_constant<int, MINE>{});
  } else {
#pragma unroll
    for (int d = 0; d < DT; d++) res[d] = o[d];
  }

  Args z = arguments();
  float l_tot = pair_sum(l_run);
  if constexpr (PAGED) {
    // (a page that is not in the cache may be some rows' only: all of the block come out as NaN, and where some do not see
    // it they are computed again below)
    int any = 0;
#pragma unroll
    for (int i = 0; i < 4 * GROUPS; i++) any |= lost_keys[i];
    if (any) l_tot = NAN;
  }
  const int col0 = group * (32 * MINE);
  if (!SHARED || parts == 1) {
    // out[row][32d + 8i + 4g + j] = res[d][4i + j] / l, by way of LDS, so that whole rows are stored
    constexpr int PITCH = ROWB / GROUPS + 16, CHUNKS = CPR / GROUPS;
    static_assert(EXCHANGE + 4 * 32 * PITCH <= 4 * TILE, "the output's slots fit the LDS");
    unsigned char* const slot = sm + EXCHANGE + w * (32 * PITCH);
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
    float zero[2] = {0.0f, 0.0f};  // (NaN behind a result that is not finite)
#pragma unroll
    for (int d = 0; d < MINE; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        half4_t h;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          h[j] = (half_t)(res[d][4 * i + j] * inv);
          zero[j & 1] = fmaf((float)h[j], 0.0f, zero[j & 1]);
        }
        *(half4_t*)(slot + frow * PITCH + (32 * d + 8 * i + 4 * g) * 2) = h;
      }
    bool finite = zero[0] + zero[1] == 0.0f;
    if (__ballot(!finite)) {
      finite = true;
#pragma unroll
      for (int d = 0; d < MINE; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          half4_t h;
          const float4_t v = {res[d][4 * i], res[d][4 * i + 1], res[d][4 * i + 2], res[d][4 * i + 3]};
          finite &= round_means(h, v, inv);
          *(half4_t*)(slot + frow * PITCH + (32 * d + 8 * i + 4 * g) * 2) = h;
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the slot is the wavefront's own)
    constexpr int RPI = 64 / CHUNKS;  // rows of a store instruction
    const int r0 = lane / CHUNKS, col = lane % CHUNKS * 8;
    int token = row_of_list(z, list0 + r0), head = list0 + r0 - token * z.group;  // of the group
    const int more_tokens = row_of_list(z, RPI), more_heads = RPI - more_tokens * z.group;
    half_t* const out = z.out + (int64_t)(hk * z.group) * z.so_z + (int64_t)q.row0 * z.so_y + col0 + col;
#pragma unroll
    for (int i = 0; i < 32 / RPI; i++) {
      if (i * RPI >= wave_rows) break;
      const int r = r0 + i * RPI;
      if (r < wave_rows && col0 + col < z.d)
        *(half8_t*)(out + (int64_t)head * z.so_z + (int64_t)token * z.so_y) = *(const half8_t*)(slot + r * PITCH + col * 2);
      token += more_tokens, head += more_heads;
      if (head >= z.group) head -= z.group, token++;
    }
    // Rows that are computed again, a group's columns of them.
    const uint64_t wrong = __ballot(!finite), far = __ballot(is_far(m_run));
    if ((wrong | far) && wave_rows > 0) {
      uint32_t again = (uint32_t)far | (uint32_t)(far >> 32);
      const uint32_t bad = (uint32_t)wrong | (uint32_t)(wrong >> 32);
      if (bad && q.rows > 1 && z.mask == ADR_MASK_CAUSAL &&
          hidden_reaches(z, q, hk, end_of_row(z, q, row_of_list(z, list0 + min(__builtin_ctz(bad), wave_rows - 1))),
                         end_of_row(z, q, row_of_list(z, block * ROWS + rows - 1)), lane))
        again |= bad;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (behind the stores above)
      for (int r = 0; r < wave_rows; r++)
        if (again >> r & 1)
          row_by_wave(arguments(), q, (list0 + r) / z.group, hk * z.group + (list0 + r) % z.group, lane, col0, col0 + 32 * MINE);
    }
  } else if (frow < wave_rows) {
    const int64_t prow = ((int64_t)(slot0 + part) * z.kv_heads + hk) * ROWS + w * 32 + frow;
    float* const po = z.part_o + prow * HD + col0 + 4 * g;
#pragma unroll
    for (int d = 0; d < MINE; d++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float4_t v;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = res[d][4 * i + j];
        *(float4_t*)(po + 32 * d + 8 * i) = v;
      }
    if (g == 0 && group == 0) z.part_ml[prow] = make_float2(m_run, l_tot);
  }
}

// Sums the parts of the blocks that lie in several workgroups' stretches, in order: a workgroup to a seam, a thread to 4
// columns of a row, as many rows at once as 256 threads have.
template <int HD, int ROWS>
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
  if (bad && b.q.rows > 1 && a.mask == ADR_MASK_CAUSAL &&
      hidden_reaches(a, b.q, hk, end_of_row(a, b.q, row_of_list(a, b.block * ROWS + r0 + __builtin_ctz(bad))),
                     end_of_row(a, b.q, row_of_list(a, b.block * ROWS + rows - 1)), lane))
    again |= bad;
  for (int x = tid >> 6; x < AT_ONCE; x += 4)
    if (again >> x & 1) {
      const int lr = b.block * ROWS + r0 + x;
      row_by_wave(arguments(), b.q, lr / a.group, hk * a.group + lr % a.group, lane);
    }
}

}  // namespace

// ---- the choice ---------------------------------------------------------------------------------------------

namespace {

int page_shift(int page_size) { return page_size >= 16 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1; }

// What the matrix-core kernels take: whole chunks of 16 bytes at 16-byte addresses, 16 key rows within the reach of a
// descriptor's 32-bit offsets, rows that do not overlap (a row behind the last key is told by its offset).
bool chunks(const SequencesArgs& a) {
  const uintptr_t ptrs = (uintptr_t)a.out | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const int64_t strides = (int64_t)a.so_y | a.so_z | a.sq_y | a.sq_z | a.sk.y | a.sk.z | a.sk.p | a.sv.y | a.sv.z | a.sv.p;
  auto near = [&](int64_t y) { return y >= a.d && y < 1 << 24; };
  return a.d % 8 == 0 && a.d <= 128 && a.so_x == 1 && a.sq_x == 1 && a.sk.x == 1 && a.sv.x == 1 && ptrs % 16 == 0 &&
         strides % 8 == 0 && strides >= 0 && near(a.sk.y) && near(a.sv.y) && (!a.table || page_shift(a.page_size) >= 0);
}

// Blocks of all key heads that there can be, and as many as a launch of 256 threads to each may have.
int64_t most_blocks(const SequencesArgs& a, int rows) {
  return ((int64_t)a.rows * a.group / rows + std::min(a.rows, a.sequences)) * a.kv_heads;
}
constexpr int64_t LAUNCH_BLOCKS = 0x7fffffff / 256;

}  // namespace

SequencesPlan sequences_plan(const SequencesArgs& a, int cus, int64_t avail) {
  SequencesPlan p = {SequencesPlan::ANY_LAYOUT, 0, 0, 0, 0, 0};
  if (!chunks(a)) return p;
  const int longest_rows = a.longest_rows > 0 ? std::min(a.longest_rows, a.rows) : a.rows;
  p.kind = (int64_t)longest_rows * a.group <= FEW ? SequencesPlan::FEW_ROWS : SequencesPlan::TILES;
  // (1: any layout; 2 ... 4: few rows; 5 ... 8: many; adr_debug_knob says which.  Other values force nothing.)
  const int forced = knob(KNOB_SEQUENCES) >= 1 && knob(KNOB_SEQUENCES) <= 8 ? knob(KNOB_SEQUENCES) : 0;
  if (forced == 1) return SequencesPlan{SequencesPlan::ANY_LAYOUT, 0, 0, 0, 0, 0};
  if (forced) p.kind = forced <= 4 ? SequencesPlan::FEW_ROWS : SequencesPlan::TILES;
  const bool few = p.kind == SequencesPlan::FEW_ROWS;
  const int rows = few ? FEW : MANY, keys = few ? FEW_KEYS : MANY_KEYS, hd = a.d <= 64 ? 64 : 128;
  const int64_t most_keys = a.table ? std::min((int64_t)a.table_width * a.page_size, (int64_t)MOST_KEYS) : a.keys;
  const double longest = a.longest > 0 ? std::min<double>(a.longest, most_keys) : most_keys;
  // Blocks of all key heads, as far as the host can tell: a sequence's last one is full by half, but where one sequence has
  // most of the rows, the others' only ones.
  const int sequences = std::min(a.rows, a.sequences);
  const double full = (double)a.rows * a.group / rows, ends = (double)longest_rows * sequences > 4.0 * a.rows ? sequences : sequences / 2.0;
  const double blocks = a.kv_heads * (few ? std::max(full, (double)sequences) : sequences <= 1 ? ceil(full) : std::max(full + ends, (double)sequences));
  p.least = 1;
  if (few) {
    // Two launches take the host and the device some 4 us more than one, and shared keys leave no workgroup with more
    // than the others.  us, fitted to 16 shapes of 12 to 32 heads, 1 to 256 sequences and 250 to 4000 keys: a block
    // by itself, four wavefronts to it, 4 + 8.5 per 1000 keys of 128 (one of 500 keys 7.8, shared 9.2; 700 9.1, 9.2; 1000
    // 14, 10.7); with more blocks than compute units the longest is a tail behind the others (100 sequences of up to 1000
    // keys, 8 key heads: 41.3, shared 43.7; up to 4000 145, 129).
    const double alone = longest * hd * 6.6e-5, all = blocks * longest * hd * 4 / 6e6;
    p.waves = blocks <= cus ? 4 : 2;
    const bool unshared = blocks <= cus ? 4.0 + alone < 9.3 + all / 2 : alone < 9.0;
    // Shared: 64 KiB of tiles in flight on a compute unit.  More only crowd each other in the caches (eight sequences of 50000 to
    // 110000 keys: two workgroups of 64 KiB to a unit 389 us, one 366), but hide the start of short stretches (256
    // sequences of up to 1000 keys: 98.8, 105).
    const int each = (hd == 64 ? 2 : 1) * (blocks >= 4.0 * cus ? 2 : 1);
    p.parts = unshared ? 0 : std::max(1, each * cus / a.kv_heads);
    if (p.parts > 0) p.waves = 2;
  } else {
    // Five ways: one or two groups of wavefronts to a block; keys shared over workgroups or not, and if so, as many as there
    // are compute units or twice that.  us, fitted to pieces of 64 to 2048 rows over 500 to 8000 keys, 8 key heads of 128
    // and 4 of 64, and to batches of pieces and tokens: start and end, a tile `one` with a compute unit to itself and `two`
    // for two tiles beside each other, of two groups or of two workgroups, and the parts' way through memory, 130 KB for a
    // workgroup.  (1024 rows over 8025 keys, 256 blocks: a group 144, two 134, shared 143; 512 rows: 122, 99, shared by
    // two groups 78, by twice as many single ones 79; 256 rows: 117, 95, 47.5, 50.5; 64 rows, shared by two groups 27.9, by
    // as many single ones 25.3.)
    const double one = hd == 64 ? 0.67 : 1.1, two = hd == 64 ? 1.02 : 2.0, way = hd == 64 ? 0.012 : 0.018;
    // (several sequences: taken to be three quarters as long as the longest)
    const double tiles = longest / MANY_KEYS + 1, work = blocks * tiles * (a.sequences == 1 ? 1.0 : 0.75);
    double best = 7 + (blocks <= cus ? one : two) * tiles;
    p.waves = 4, p.parts = 0;
    p.least = 4;
    if (blocks <= cus && 8 + two * tiles / 2 < best) best = 8 + two * tiles / 2, p.waves = 8;
    auto shared = [&](int waves, double most, double start, double tile) {
      double n = std::min(most, sqrt(work * tile / way));
      // (the blocks of one sequence are of one size, and go into equally many parts; of several, one goes into half a part
      // too few in the mean)
      if (a.sequences == 1) n = floor(n / blocks) * blocks;
      if (a.sequences > 256 || n < (a.sequences == 1 ? 2.0 : 1.5) * blocks) return;
      const double us = start + work * tile / (a.sequences == 1 ? n : n - blocks / 2) + n * way;
      if (us < best) best = us, p.waves = waves, p.parts = (int)(n / a.kv_heads + 0.5);
    };
    shared(4, cus * 15 / 16.0, 12, one);  // (with as many as there are units some share one: 26.0, 240 of them 24.8)
    shared(4, 2.0 * cus, 12, two);
    shared(8, cus, 14, two / 2);
  }
  if (forced) {  // (shared in small parts, so that short sequences are divided too)
    const bool divides = forced == 4 || (forced > 6 && a.sequences <= 256 && full + sequences < 1000);
    p.waves = forced == 3 || forced == 5 || forced == 7 ? 4 : forced == 6 || forced == 8 ? 8 : 2;
    p.parts = divides ? std::max(16, cus / a.kv_heads) : 0;
    p.least = 1;
  }
  // (pieces grow where there could be more of them than the line counts)
  const double most_tiles = ((double)a.rows * a.group / rows + a.sequences) * (most_keys / keys + 2.0);
  for (p.shift = FEW_SHIFT; most_tiles > ldexp(0x1p29, p.shift) && p.shift < 25; p.shift++) {}
  // (slots: two to a stretch of few rows, one to a part of many)
  const int64_t part = ((few ? 2 : 1) * (int64_t)rows * (hd * 4 + 8) + (int64_t)sizeof(Seam)) * a.kv_heads;
  p.parts = (int)std::min<int64_t>(p.parts, avail / part);
  if (p.parts < 2) p.parts = 0;
  // (hundreds of thousands of sequences with a block to each: the kernel whose wavefronts take one row after the other)
  if (p.parts == 0 && most_blocks(a, rows) > LAUNCH_BLOCKS) return SequencesPlan{SequencesPlan::ANY_LAYOUT, 0, 0, 0, 0, 0};
  p.workspace_bytes = p.parts * part;
  return p;
}

template <int HD, bool PAGED>
static hipError_t launch_blocks(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  const bool few = p.kind == SequencesPlan::FEW_ROWS;
  const int rows = few ? FEW : MANY;
  Job job;
  (SequencesArgs&)job = a;
  job.page_shift = PAGED ? page_shift(a.page_size) : 0;
  job.parts = p.parts, job.shift = p.shift, job.least = p.least;
  job.part_o = (float*)workspace;
  job.per_head = 1.0 / a.group;
  const int64_t part_rows = (int64_t)(few ? 2 : 1) * p.parts * a.kv_heads * rows;
  job.part_ml = (float2*)(job.part_o + (p.parts > 0 ? part_rows * HD : 0));
  job.seams = (Seam*)(job.part_ml + (p.parts > 0 ? part_rows : 0));
  // Unshared: as many as there can be blocks.  Shared: a stretch to each, or a part.
  const int64_t most = most_blocks(a, rows), shared = (int64_t)p.parts * a.kv_heads;
  const int64_t blocks = p.parts == 0 ? most : few ? shared : std::max(shared, most);
  if (blocks > LAUNCH_BLOCKS) return hipErrorInvalidConfiguration;
  const int at_once = std::min(rows, 1024 / HD);  // rows of the joining workgroups
  const dim3 grid((unsigned)blocks), join((unsigned)((few ? p.parts - 1 : p.parts / 2) * a.kv_heads * (rows / at_once)));
  const dim3 threads(64 * p.waves);
  const size_t few_lds = (size_t)p.waves * 4 * FEW_KEYS * HD * 2;
  if (few && p.parts > 0) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 2, true>), grid, threads, few_lds, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, FEW>), join, dim3(256), 0, stream, job);
  } else if (few && p.waves == 2) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 2, false>), grid, threads, few_lds, stream, job);
  } else if (few) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 4, false>), grid, threads, few_lds, stream, job);
  } else if (p.parts > 0) {
    if (p.waves == 8) hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, true, 2>), grid, threads, 0, stream, job);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, true, 1>), grid, threads, 0, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, MANY>), join, dim3(256), 0, stream, job);
  } else if (p.waves == 8) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, false, 2>), grid, threads, 0, stream, job);
  } else {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, false, 1>), grid, threads, 0, stream, job);
  }
  return hipGetLastError();
}

hipError_t launch_attention_sequences(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  if (p.kind == SequencesPlan::ANY_LAYOUT) {
    const int64_t waves = (int64_t)a.rows * a.heads;
    const int64_t grid = std::min<int64_t>((waves + 3) / 4, 1 << 22);
    Job job = {};
    (SequencesArgs&)job = a;
    hipLaunchKernelGGL(attention_any_layout_kernel, dim3((unsigned)grid), dim3(256), 0, stream, job);
    return hipGetLastError();
  }
  if (a.d <= 64) return a.table ? launch_blocks<64, true>(stream, a, p, workspace) : launch_blocks<64, false>(stream, a, p, workspace);
  return a.table ? launch_blocks<128, true>(stream, a, p, workspace) : launch_blocks<128, false>(stream, a, p, workspace);
}

}  // namespace adr
