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

constexpr float NO_SCORE = -1.0e30f;  // below any score of finite operands; exp2(-inf - NO_SCORE) is 0, not NaN

// A sequence's rows and keys.
struct Sequence {
  int index, row0, rows;  // first row of the [heads, rows, d] views
  int key0, keys;         // first key of packed ones
};

__device__ __forceinline__ Sequence sequence_at(const SequencesArgs& a, int s) {
  Sequence q;
  q.index = s;
  q.row0 = clamp_to(a.row_offsets[s], a.rows);
  q.rows = max(clamp_to(a.row_offsets[s + 1], a.rows) - q.row0, 0);
  if (a.table) {
    q.key0 = 0;
    const int64_t room = min((int64_t)a.table_width * a.page_size, (int64_t)MOST_KEYS);
    q.keys = (int)min((int64_t)max(a.keys_of[s], 0), room);
  } else {
    q.key0 = clamp_to(a.keys_of[s], a.keys);
    q.keys = max(clamp_to(a.keys_of[s + 1], a.keys) - q.key0, 0);
  }
  return q;
}

// Key x of the sequence as element offsets of its key and value rows (head 0); false: on no page of the cache.
__device__ __forceinline__ bool key_at(const SequencesArgs& a, const Sequence& q, int x, int64_t& k, int64_t& v) {
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
// and a lane to every 64th column for the sums.  Only keys that the row sees are read.  Probabilities stay in 32 bits.
constexpr int GENERAL_MAX_D = 256;
__device__ __forceinline__ void row_by_wave(const SequencesArgs& a, const Sequence& q, int j, int h, int lane) {
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
      s = good ? s * a.c : NAN;
    }
    float top = s;
    for (int i = 32; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));  // (not the NaNs)
    const float m_new = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    const float p = __builtin_amdgcn_exp2f(s - m);
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
    if (c * 64 + lane < a.d) O[(c * 64 + lane) * (int64_t)a.so_x] = (half_t)(o[c] * inv);
}

// Any layout: a wavefront per row and query head.
__global__ __launch_bounds__(256) void attention_any_layout_kernel(SequencesArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t i = (int64_t)blockIdx.x * 4 + wave; i < (int64_t)a.rows * a.heads; i += (int64_t)gridDim.x * 4) {
    const int h = (int)(i / a.rows), row = (int)(i - (int64_t)h * a.rows);
    const Sequence q = sequence_at(a, sequence_of_row(a.row_offsets, a.sequences, row, lane));
    if (row < q.row0 || row >= q.row0 + q.rows) continue;
    row_by_wave(a, q, row - q.row0, h, lane);
  }
}


// ---- who does what -----------------------------------------------------------------------------------
//
// The rows of a sequence times the query heads of a group, R = rows * group, are one list (row of the sequence
// first, head of the group second), cut into blocks of ROWS: the heads of a group share every key that is read.
// A workgroup takes one block of one key head, or one of several parts of its keys.  The host knows neither
// the sequences' rows nor their keys, only how many workgroups fill the chip (`parts` for each key head), so the
// division is made on the device, by every wavefront for itself and with the same result: with W the sum over all
// blocks of their key tiles, no workgroup gets more than C = max(W / parts, min_steps) tiles, and a block
// with more is divided evenly.  That is at most parts + blocks workgroups, and no sequence, however long among
// short ones, holds up the others.  Divided blocks have their parts' results in consecutive slots of the workspace,
// fewer than 2 * parts of them (each has more than C tiles, and there are W in all).
struct Share {
  int parts, min_steps;  // 0: nothing is divided
  float* part_o;         // [slot][key head][ROWS][HD] unnormalised sums
  float2* part_ml;       // [slot][key head][ROWS] (maximum in log2 units, sum)
};

struct Piece {
  Sequence q;
  int block;          // of the sequence's rows
  int part, parts;    // of its keys
  int slot;           // of the first part's results
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

// Piece number `index` of the list above (DIVIDED: block number `index` of those that are divided); false: there are
// fewer.  A lane takes 4 sequences of 256.
template <int ROWS, int KEYS, bool DIVIDED>
__device__ __forceinline__ bool find_piece(const SequencesArgs& a, const Share& share, int index, int lane, Piece& piece) {
  constexpr int EACH = 4;
  int blocks[EACH], tiles[EACH];
  auto load = [&](int base) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      const int s = base + lane * EACH + e;
      blocks[e] = tiles[e] = 0;
      if (s < a.sequences) {
        const Sequence q = sequence_at(a, s);
        blocks[e] = (int)(((int64_t)q.rows * a.group + ROWS - 1) / ROWS);
        tiles[e] = (q.keys + KEYS - 1) / KEYS;
      }
    }
  };
  load(0);
  int most = 0x7fffffff;  // C
  if (share.parts > 0) {
    // (in 32-bit floats: the sum need not be exact, only the same everywhere)
    float work = 0.0f;
    for (int base = 0;;) {
#pragma unroll
      for (int e = 0; e < EACH; e++) work += (float)blocks[e] * (float)tiles[e];
      base += 64 * EACH;
      if (base >= a.sequences) break;
      load(base);
    }
    for (int i = 1; i < 64; i <<= 1) work += __shfl_xor(work, i);
    most = max(share.min_steps, (int)fminf(ceilf(work / (float)share.parts), 1.0e9f));
    if (a.sequences > 64 * EACH) load(0);
  }
  int slot = 0;
  for (int base = 0; base < a.sequences;) {
    int count[EACH], parts[EACH], sum = 0, slots = 0;
#pragma unroll
    for (int e = 0; e < EACH; e++) {
      parts[e] = tiles[e] <= most ? 1 : (tiles[e] + most - 1) / most;
      const int divided = parts[e] > 1 ? blocks[e] : 0;
      count[e] = DIVIDED ? divided : blocks[e] * parts[e];
      sum += count[e];
      slots += divided * parts[e];
    }
    const int upto = add_scan(sum), slots_upto = add_scan(slots);
    const uint64_t behind = __ballot(upto > index);
    if (behind) {
      const int at = __builtin_ctzll(behind);
      int i = index - (__shfl(upto, at) - __shfl(sum, at));
      slot += __shfl(slots_upto, at) - __shfl(slots, at);
#pragma unroll
      for (int e = 0; e < EACH; e++) {
        const int n = __shfl(count[e], at), p = __shfl(parts[e], at), b = __shfl(blocks[e], at);
        if (i < n) {
          // (the last blocks first: under the mask they have the most keys)
          const int block = b - 1 - (DIVIDED ? i : i / p);
          piece.q = sequence_at(a, base + at * EACH + e);
          piece.block = block;
          piece.parts = p;
          piece.part = DIVIDED ? 0 : i % p;
          piece.slot = slot + (b - 1 - block) * p;
          return true;
        }
        i -= n;
        if (p > 1) slot += b * p;
      }
    }
    index -= __shfl(upto, 63);
    slot += __shfl(slots_upto, 63);
    base += 64 * EACH;
    if (base < a.sequences) load(base);
  }
  return false;
}

// One past the last key that some row of the block sees, and of one row.
__device__ __forceinline__ int end_of_row(const SequencesArgs& a, const Sequence& q, int j) {
  return a.mask == ADR_MASK_CAUSAL ? clamp_to(j + q.keys - q.rows + 1, q.keys) : q.keys;
}

// Pages of 2^shift slots, 16 at least: 16 keys from a multiple of 16 on lie on one page, so that a transfer of 16 rows
// has one base address.
struct Pages {
  int shift;
};

// ---- few rows: generation, a few tokens at once ----------------------------------------------------------
//
// A block of 16 rows against its keys: a read of the keys and values.  The workgroup's wavefronts walk tiles of
// 32 keys in turn, each through two tiles' worth of LDS of its own, so that the loop has no barrier.  S^T = K Q^T, so
// that a lane holds scores of one row, and O^T = V^T P^T, on MFMA 16x16x32; probabilities are rounded to fp16, the
// matrix cores' operands, sums and scores stay in 32 bits.
template <int HD, bool PAGED, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attention_few_rows_kernel(SequencesArgs a, Share share, Pages pages) {
  constexpr int CPR = HD / 8, KEYS = 32, ROWS = 16;
  constexpr int ROWB = HD * 2, TILE = KEYS * ROWB;  // bytes of a tile row, of a K or V tile
  constexpr int NI = TILE / 1024;                   // transfers per tile
  constexpr int KS = HD / 32, DB = HD / 16;         // k-steps of S, blocks of 16 output columns
  constexpr int WAVE = 4 * TILE;                    // K0 K1 V0 V1 of a wavefront
  constexpr int PITCH = HD + 4;                     // of the partial results' rows, in floats
  constexpr int BIAS = 1024;                        // bytes that descriptors start ahead, so that no offset is negative
  static_assert(16 * (PITCH + 2) * 4 + 16 <= WAVE, "the partial results fit the tiles' LDS");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[WAVES * WAVE];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int frow = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % a.kv_heads;
  Piece pc;
  if (!find_piece<ROWS, KEYS, false>(a, share, blockIdx.x / a.kv_heads, lane, pc)) return;
  const Sequence q = {__builtin_amdgcn_readfirstlane(pc.q.index), __builtin_amdgcn_readfirstlane(pc.q.row0),
                      __builtin_amdgcn_readfirstlane(pc.q.rows), __builtin_amdgcn_readfirstlane(pc.q.key0),
                      __builtin_amdgcn_readfirstlane(pc.q.keys)};
  const int block = __builtin_amdgcn_readfirstlane(pc.block), part = __builtin_amdgcn_readfirstlane(pc.part),
            parts = __builtin_amdgcn_readfirstlane(pc.parts), slot0 = __builtin_amdgcn_readfirstlane(pc.slot);
  const int rows = min(ROWS, q.rows * a.group - block * ROWS);          // of the block
  const int list_row = block * ROWS + min(frow, rows - 1), row = list_row / a.group, gh = list_row - row * a.group;

  const int last_end = end_of_row(a, q, (block * ROWS + rows - 1) / a.group);  // of the block's last row
  const int all = (last_end + KEYS - 1) / KEYS;
  const int tile0 = (int)((int64_t)all * part / parts), tile1 = (int)((int64_t)all * (part + 1) / parts);
  const int row_end = min(last_end, tile1 * KEYS);
  const int tiles = max(0, (tile1 - tile0 - w + WAVES - 1) / WAVES);  // of this wavefront: tile0 + w + WAVES i

  const half_t* const K = a.k + hk * a.sk.z + (PAGED ? 0 : q.key0 * a.sk.y);
  const half_t* const V = a.v + hk * a.sv.z + (PAGED ? 0 : q.key0 * a.sv.y);
  const uint32_t lds0 = (uint32_t)(uintptr_t)ADR_LDS_PTR(smem) + w * WAVE;
  const unsigned char* const sm = smem + w * WAVE;
  // Byte offsets of a lane's chunks in 16 rows (the second 16 rows of a tile repeat them); chunks behind the head
  // dimension lie behind every descriptor's end and come as zeros.
  uint32_t koff[NI / 2], voff[NI / 2];
#pragma unroll
  for (int j = 0; j < NI / 2; j++) {
    int krow, kc;
    k_chunk_inv<CPR>(j * 64 + lane, krow, kc);
    const int vrow = (j * 64 + lane) / CPR, vc = (lane % CPR) ^ v_swz8<CPR>(vrow);
    koff[j] = kc * 8 < a.d ? (uint32_t)((krow * (int)a.sk.y + kc * 8) * 2 + BIAS - (j & 1) * 1024) : 0x7fff0000u;
    voff[j] = vc * 8 < a.d ? (uint32_t)((vrow * (int)a.sv.y + vc * 8) * 2 + BIAS - (j & 1) * 1024) : 0x7fff0000u;
  }
  // The pages of 32 of the wavefront's tiles at a time, a lane to each 16 keys.
  int page = 0;
  bool lost = false;  // a key's page is not in the cache
  auto look_up = [&](int i) __attribute__((always_inline)) {
    const int key = (tile0 + w + WAVES * (i + (lane >> 1))) * KEYS + 16 * (lane & 1);
    page = 0;
    if (key < row_end) {
      page = a.table[(int64_t)q.index * a.table_pitch + (key >> pages.shift)];
      if (page < 0 || page >= a.pages) lost = true, page = -1;
    }
  };
  auto fetch = [&](int i) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int key = (tile0 + w + WAVES * i) * KEYS + 16 * h;
      int left = min(row_end - key, 16);
      int64_t ko, vo;
      if constexpr (PAGED) {
        const int p = __builtin_amdgcn_readlane(page, 2 * (i & 31) + h), slot = key & ((1 << pages.shift) - 1);
        if (p < 0) left = 0;
        ko = p * a.sk.p + slot * a.sk.y;
        vo = p * a.sv.p + slot * a.sv.y;
      } else {
        ko = key * a.sk.y;
        vo = key * a.sv.y;
      }
      const uint64_t pk = (uint64_t)(K + ko) - BIAS, pv = (uint64_t)(V + vo) - BIAS;
      const u32x4_t dk = {(uint32_t)pk, (uint32_t)(pk >> 32) & 0xffffu,
                          left > 0 ? (uint32_t)(((left - 1) * (int)a.sk.y + a.d) * 2 + BIAS) : 0u, 0x00020000u};
      const u32x4_t dv = {(uint32_t)pv, (uint32_t)(pv >> 32) & 0xffffu,
                          left > 0 ? (uint32_t)(((left - 1) * (int)a.sv.y + a.d) * 2 + BIAS) : 0u, 0x00020000u};
#pragma unroll
      for (int j = 0; j < NI / 2; j += 2)
        dma_buffer_pair<0>(lds0 + (i & 1) * TILE + (h * (NI / 2) + j) * 1024, koff[j], koff[j + 1], dk);
#pragma unroll
      for (int j = 0; j < NI / 2; j += 2)
        dma_buffer_pair<0>(lds0 + (2 + (i & 1)) * TILE + (h * (NI / 2) + j) * 1024, voff[j], voff[j + 1], dv);
    }
  };

  if constexpr (PAGED) look_up(0);
  half8_t qf[KS];
  const half_t* const qrow =
      a.q + (int64_t)(hk * a.group + gh) * a.sq_z + (int64_t)(q.row0 + row) * a.sq_y;
#pragma unroll
  for (int ks = 0; ks < KS; ks++) {
    const int col = ks * 32 + g * 8;
    qf[ks] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    if (col < a.d) qf[ks] = *(const half8_t*)(qrow + col);
  }
  // (the loads above have landed before the transfers' own count begins)
#pragma unroll
  for (int ks = 0; ks < KS; ks++) asm volatile("" : "+v"(qf[ks]));
  if (tiles > 0) fetch(0);
  if (tiles > 1) fetch(1);
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
  // Tile i; `next`: there is a tile i + 1, `more`: and a tile i + 2.
  auto tile = [&](int i, auto next, auto more) __attribute__((always_inline)) {
    wait_vm<decltype(next)::value ? 2 * NI : 0>();  // tile i has landed (tile i + 1 may be in flight)
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
    half8_t vf[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) {
      const unsigned char* const p0 = cV + offV[db];
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0 + 16 * ROWB));
      vf[db] = __builtin_shufflevector(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, hi),
                                       0, 1, 2, 3, 4, 5, 6, 7);
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
    const float m_new = fmaxf(m_run, fmaxf(x, y) * a.c), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    float sum = 0.0f;
    u32x4_t pf;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float2_t e;
#pragma unroll
        for (int j = 0; j < 2; j++) e[j] = __builtin_amdgcn_exp2f(fmaf(s[kb][r + j], a.c, -m_new));
        sum += e[0] + e[1];
        pf[kb * 2 + r / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(e, half2_t));
      }
    l_run = l_run * alpha + sum;
#pragma unroll
    for (int db = 0; db < DB; db++) {
      o[db] *= alpha;
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[db], __builtin_bit_cast(half8_t, pf), o[db], 0, 0, 0);
    }
    // (the tile has been read: its fragments are in registers)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (decltype(more)::value) {
      if constexpr (PAGED) {
        if (((i + 2) & 31) == 0) look_up(i + 2);
      }
      fetch(i + 2);
    }
  };
  const std::true_type yes{};
  const std::false_type no{};
  int i = 0;
  for (; i + 2 < tiles; i++) tile(i, yes, yes);
  if (i + 1 < tiles) tile(i++, yes, no);
  if (i < tiles) tile(i, no, no);

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
    if (parts == 1) {
      const int lr = block * ROWS + r, token = lr / a.group, h = hk * a.group + lr - token * a.group;
      half4_t v;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      bool finite = true;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        finite = finite && fabsf(sum[j] * inv) < INFINITY;
        v[j] = (half_t)(sum[j] * inv);
      }
      if (!finite) atomicOr(bad_rows, 1 << r);
      if (col < a.d)
        *(half4_t*)(a.out + (int64_t)h * a.so_z + (int64_t)(q.row0 + token) * a.so_y + col) = v;
    } else {
      const int64_t prow = ((int64_t)(slot0 + part) * a.kv_heads + hk) * ROWS + r;
      *(float4_t*)(share.part_o + prow * HD + col) = sum;
      if (col == 0) share.part_ml[prow] = make_float2(m_all, l);
    }
  }
  // A value that is no number times the zero of a key that the row does not see is no zero: such rows are computed
  // again from the keys that they see.
  if (parts == 1 && q.rows > 1 && a.mask == ADR_MASK_CAUSAL) {
    __syncthreads();
    for (int r = w; r < rows; r += WAVES)
      if (*bad_rows >> r & 1) {
        const int lr = block * ROWS + r;
        row_by_wave(a, q, lr / a.group, hk * a.group + lr % a.group, lane);
      }
  }
}

// Sums the parts of a divided block: a wavefront to a row, 16 rows to a workgroup, HD / 64 columns to a lane; parts in order.
template <int HD, int ROWS, int KEYS>
__global__ __launch_bounds__(256) void attention_join_kernel(SequencesArgs a, Share share) {
  constexpr int C = HD / 64;
  typedef float vec_t __attribute__((ext_vector_type(C)));
  typedef half_t hvec_t __attribute__((ext_vector_type(C)));
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int hk = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads;
  constexpr int GROUPS = ROWS / 16;
  Piece pc;
  if (!find_piece<ROWS, KEYS, true>(a, share, rest / GROUPS, lane, pc)) return;
  const int rows = min(ROWS, pc.q.rows * a.group - pc.block * ROWS);
  for (int r = rest % GROUPS * 16 + w; r < min(rows, rest % GROUPS * 16 + 16); r += 4) {
    const int64_t first = ((int64_t)pc.slot * a.kv_heads + hk) * ROWS + r, step = (int64_t)a.kv_heads * ROWS;
    vec_t acc = 0.0f;
    float m = NO_SCORE, l = 0.0f;
    for (int s0 = 0; s0 < pc.parts; s0 += 64) {
      const float2 ml = s0 + lane < pc.parts ? share.part_ml[first + (s0 + lane) * step] : make_float2(NO_SCORE, 0.0f);
      float top = ml.x;
      for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
      const float m_new = fmaxf(m, top), alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      const float f = __builtin_amdgcn_exp2f(ml.x - m);
      float sum = ml.y * f;
      for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
      l = l * alpha + sum;
      acc *= alpha;
      const int n = min(64, pc.parts - s0);
      for (int s = 0; s < n; s += 8) {
        vec_t v[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
          v[j] = *(const vec_t*)(share.part_o + (first + (s0 + min(s + j, n - 1)) * step) * HD + lane * C);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float fj = __shfl(f, s + j);
          if (s + j < n) acc += v[j] * fj;
        }
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    acc *= inv;
    const int lr = pc.block * ROWS + r, token = lr / a.group, h = hk * a.group + lr - token * a.group;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < C; j++) finite = finite && fabsf(acc[j]) < INFINITY;
    if (__ballot(!finite) && pc.q.rows > 1 && a.mask == ADR_MASK_CAUSAL) {
      row_by_wave(a, pc.q, token, h, lane);
      continue;
    }
    if (lane * C < a.d)
      *(hvec_t*)(a.out + (int64_t)h * a.so_z + (int64_t)(pc.q.row0 + token) * a.so_y + lane * C) =
          __builtin_convertvector(acc, hvec_t);
  }
}

}  // namespace

// ---- the choice ---------------------------------------------------------------------------------------------

namespace {

constexpr int FEW = 16, FEW_KEYS = 32, FEW_WAVES = 2;
// (a few more than the division above can come to: its sum of work is rounded)
constexpr int SPARE = 8;

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

int64_t slot_bytes(int rows, int hd) { return (int64_t)rows * (hd * 4 + 8); }

}  // namespace

SequencesPlan sequences_plan(const SequencesArgs& a, int cus, int64_t avail) {
  SequencesPlan p = {SequencesPlan::ANY_LAYOUT, 0, 0, 0};
  if (!chunks(a)) return p;
  p.kind = SequencesPlan::FEW_ROWS;
  const int hd = a.d <= 64 ? 64 : 128;
  const int64_t slot = slot_bytes(FEW, hd) * a.kv_heads;
  p.parts = std::max(1, 2 * cus / a.kv_heads);
  p.parts = (int)std::max<int64_t>(0, std::min<int64_t>(p.parts, (avail / slot - SPARE) / 2));
  p.min_steps = 8;
  p.workspace_bytes = p.parts > 0 ? (2 * p.parts + SPARE) * slot : 0;
  return p;
}

template <int HD, bool PAGED>
static hipError_t launch_few_rows(hipStream_t stream, const SequencesArgs& a, const Share& share) {
  const Pages pages = {PAGED ? page_shift(a.page_size) : 0};
  const int64_t blocks = (int64_t)a.rows * a.group / FEW + a.sequences + share.parts + SPARE;  // at most
  if (blocks * a.kv_heads > 0x7fffffff / (64 * FEW_WAVES)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, FEW_WAVES>), dim3((unsigned)(blocks * a.kv_heads)),
                     dim3(64 * FEW_WAVES), 0, stream, a, share, pages);
  if (share.parts > 0)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, FEW, FEW_KEYS>), dim3((unsigned)(share.parts * a.kv_heads)),
                       dim3(256), 0, stream, a, share);
  return hipGetLastError();
}

hipError_t launch_attention_sequences(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  if (p.kind == SequencesPlan::ANY_LAYOUT) {
    const int64_t waves = (int64_t)a.rows * a.heads;
    const int64_t grid = std::min<int64_t>((waves + 3) / 4, 1 << 22);
    hipLaunchKernelGGL(attention_any_layout_kernel, dim3((unsigned)grid), dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  const int hd = a.d <= 64 ? 64 : 128;
  Share share = {p.parts, p.min_steps, (float*)workspace, nullptr};
  if (p.parts > 0) share.part_ml = (float2*)((float*)workspace + ((int64_t)2 * p.parts + SPARE) * a.kv_heads * FEW * hd);
  if (a.table) return hd == 128 ? launch_few_rows<128, true>(stream, a, share) : launch_few_rows<64, true>(stream, a, share);
  return hd == 128 ? launch_few_rows<128, false>(stream, a, share) : launch_few_rows<64, false>(stream, a, share);
}

}  // namespace adr
