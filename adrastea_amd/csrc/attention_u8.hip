// Attention over a paged cache in 8 bits: code c of key x stands for (c - 127.5) ks[x], of its value for (c - 127.5) vs[x].
//
//   s[x] = <q, K[x] - 127.5> ks[x],   out = sum_x w[x] (V[x] - 127.5) / sum_x softmax weights,   w[x] = weight of x times vs[x]
//
// The matrix cores are given the codes as they are: a byte, widened, is the fp16 number c 2^-24, exact, and below the normal
// numbers, which are not flushed.  So scores are 32-bit sums of exact products that begin at -127.5 sum(q) and are multiplied by the
// key's scale once; a value's scale goes into the probability, the only thing that is rounded, and 127.5 times the sum of the
// rounded probabilities (one more product, with ones) is taken off the sums of values: at the end, and every 16 tiles, so that what it leaves
// of their 32 bits does not shrink with the context.  (Values of 16 codes around the middle, as where one large value of a head sets its
// scale, over 24000 keys: with the offset in all of the sums their means were off by 3 to 21 times the last rounding to fp16.  What is left is
// half of that rounding, from the sums within an instruction.  128 sequences of 3 to 4000 keys 113.9 us -> 114.4, others as before.)
//
// Few rows round it to two fp16 numbers, the second what the first leaves: 22 bits.  Results are then off by 0.00021 of their root mean
// square, which is the last rounding to fp16; with one number it was 0.00025 to 0.00032.  The matrix cores have room for the second
// product (us, with one -> with both: a batch of tokens 51.3 -> 52.0, long contexts 200.9 -> 202.1, one user 11.5 -> 11.7, drafts 44.3 ->
// 44.9).  Many rows round it to one: 0.00028, as values in 16 bits have it.  The loop has no registers for the other, which goes
// through scratch: a prompt's piece 167 -> 274 us, one user's draft 26.8 -> 35.5.
//
// What is kept within fp16's range is thus the probability times the value's scale: a row's reference follows the largest
// s c + log2 vs, as attention_sequences.hip says of s c, with vs taken as 2^-25 where it is less (a key of such values may have
// all the weight; then the others' part of the result is below fp16's numbers).
// A key whose scales are no numbers of the format, or which is on no page, has NaN for a key's scale and 0 for a value's: rows that see
// it become NaN, and to the others it is a finite value of weight 0.
//
// Who does what, the softmax and the parts that are joined are those of attention_sequences.hip.
#include <algorithm>
#include <type_traits>

#include "attention_tiles.hpp"

namespace adr {
namespace {

__global__ __launch_bounds__(256) void attention_u8_any_layout_kernel(Job) { rows_one_by_one<true>(arguments()); }

// Where in a 256-byte line of the value tile a 16-byte chunk lies: the transposing reads of 32 lanes take a chunk each of rows
// 4 g ... 4 g + 3 and 16 + 4 g ... 16 + 4 g + 3 of two g, and these 16 are on different banks.
template <int CPR>
__device__ __forceinline__ int value_swizzle(int row) {
  return CPR == 8 ? ((row >> 1) & 3) | (row >> 4 & 1) << 2 : ((row >> 2) & 1) | (row >> 4 & 1) << 1;
}

// Transfers of a tile's 16 rows: 1 or 2 KiB.
template <int N>
__device__ __forceinline__ void transfer_once(uint32_t lds, const uint32_t (&voff)[N], u32x4_t desc) {
  if constexpr (N == 2) dma_buffer_once<2>(lds, voff, desc);
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                 :: "s"(lds), "v"(voff[0]), "s"(desc) : "memory");
}

// The scales of 16 keys of a page, of which `left` are there (what comes for the others does not count).
struct Scales {
  u32x4_t lo, hi;
};
__device__ __forceinline__ Scales read_scales(const half_t* p, int64_t step, bool side_by_side, int left) {
  Scales s;
  if (side_by_side) {
    s.lo = *(const u32x4_t*)p, s.hi = *(const u32x4_t*)(p + 8);
  } else {
    uint16_t v[16];
#pragma unroll
    for (int e = 0; e < 16; e++) v[e] = half_to_bits(p[min(e, left - 1) * step]);
    __builtin_memcpy(&s, v, 32);
  }
  return s;
}

// ---- few rows: generation, a few tokens or a small draft at once ---------------------------------------------
//
// A block of 16 rows against its keys, as attention_few_rows_kernel: tiles of 32 keys, two of each wavefront's in LDS.  A tile's
// codes go from LDS to registers as they are, values through the transposing read of bytes, and become fp16 there.
//
// Long contexts are bound by memory: eight sequences of 50000 to 110000 keys (40 / 8 heads of 128, 1.22 GB) 195 us, 6.2 TB/s.
// One wavefront alone takes 1.1 to 1.3 us a tile, so that blocks get eight where they
// are few: one of 777 keys (32 / 32 heads) 11.7 us, with four 12.7, with two 14.1.  64 sequences of 3 to 4000 keys (32 / 8, 251 MB)
// 51.5: a unit has two blocks one after the other, each with some 8 us before its first tile and behind its last, in which nothing
// else is on its way there (four wavefronts, two blocks beside each other, 56; two 85).  24 drafts of 2 to 13 tokens over up to 6000 keys
// 44.8 (longest sequences first; in the batch's order 59.5).
constexpr int FEW_AHEAD = 8;
constexpr int few_bytes(int hd) { return 4 * FEW_KEYS * hd + 3 * 2 * FEW_AHEAD * FEW_KEYS * 2; }  // of LDS, a wavefront

template <int HD, int WAVES, bool SHARED, bool TREE>
__global__ __launch_bounds__(64 * WAVES, 2) void attention_u8_few_rows_kernel(Job) {
  constexpr int CPR = HD / 16, KEYS = 32, ROWS = 16;
  constexpr int ROWB = HD, TILE = KEYS * ROWB;      // bytes of a tile row, of a K or V tile
  constexpr int NI = TILE / 1024;                   // transfers per tile
  constexpr int KP = HD / 64, DB = HD / 16;         // pairs of k-steps of S, blocks of 16 output columns
  constexpr int AHEAD = FEW_AHEAD;                  // tiles whose addresses are looked up at once
  constexpr int SCALES = 4 * TILE;                  // K0 K1 V0 V1 of a wavefront, then twice as many tiles' scales:
  constexpr int KIND = 2 * AHEAD * KEYS * 2;        // bytes of those of keys, of values, and of their logarithms
  constexpr int WAVE = few_bytes(HD);
  constexpr int PITCH = HD + 4;                     // of the partial results' rows, in floats
  constexpr int BIAS = NI / 2 * 1024;               // bytes that descriptors start ahead, so that no offset is negative
  static_assert(16 * (PITCH + 2) * 4 + 16 <= WAVE, "the partial results fit the tiles' LDS");
  static_assert(2 * KP * 1024 <= TILE, "the queries fit a tile of values");
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // (WAVES * WAVE bytes)

  Args first = arguments();
  early<true, !SHARED>(first);
  const int kv_heads = first.kv_heads, hk = blockIdx.x % kv_heads, wg = blockIdx.x / kv_heads;
  Roster<ROWS, KEYS, true, SHARED, !SHARED> roster;
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

  const uint32_t lds0 = (uint32_t)(uintptr_t)ADR_LDS_PTR(smem) + w * WAVE;
  unsigned char* const sm = smem + w * WAVE;
  // The queries' fragments, by way of the last tile of values: of 64 columns a lane has 16, 8 to each of two k-steps, as
  // it reads 16 codes of a key at once.  (Chunks behind the head dimension are zeros below.)
  const int d = a.d, k_stride = (int)a.sk.y, v_stride = (int)a.sv.y;
  const half_t* const qrow = a.q + (int64_t)(hk * a.group + gh) * a.sq_z + (int64_t)(q.row0 + row) * a.sq_y;
#pragma unroll
  for (int ks = 0; ks < 2 * KP; ks++) {
    const int col = (ks >> 1) * 64 + g * 16 + (ks & 1) * 8;
    dma_global(lds0 + SCALES - TILE + ks * 1024, qrow + (col < d ? col : 0));
  }
  // Byte offsets of a lane's chunks in 16 rows; chunks behind the head dimension lie behind every descriptor's end and come
  // as zeros.  Values' chunks are placed differently in the second 16 rows.
  uint32_t koff[NI / 2], voff[2][NI / 2];
#pragma unroll
  for (int j = 0; j < NI / 2; j++) {
    int krow, kc;
    k_chunk_inv<CPR>(j * 64 + lane, krow, kc);
    koff[j] = kc * 16 < d ? (uint32_t)(krow * k_stride + kc * 16 + BIAS - j * 1024) : 0x7fff0000u;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int vrow = (j * 64 + lane) / CPR, vc = (lane % CPR) ^ value_swizzle<CPR>(vrow + 16 * h);
      voff[h][j] = vc * 16 < d ? (uint32_t)(vrow * v_stride + vc * 16 + BIAS - j * 1024) : 0x7fff0000u;
    }
  }
  // Where the keys (lanes 0 ... 31) and values (32 ... 63) of AHEAD of the wavefront's tiles lie, a lane to each 16, and their
  // scales, which go to LDS.  (Code addresses are as they come; bit 63 says that there are keys.)
  const bool side_by_side = a.sks.y == 1 && a.svs.y == 1 && (a.sks.z | a.sks.p | a.svs.z | a.svs.p) % 8 == 0 &&
                            ((uintptr_t)a.k_scale | (uintptr_t)a.v_scale) % 16 == 0;
  uint32_t at_lo = 0, at_hi = 0, bad = 0;
  Scales looked_up;
  auto look_up = [&](int i) __attribute__((always_inline)) {
    Args c = arguments();
    const int t = i + (lane >> 1 & (AHEAD - 1)), key = (tile0 + w + WAVES * t) * KEYS + 16 * (lane & 1), left = row_end - key;
    const bool is_v = lane >= 32;
    uint64_t at = 0;  // (no keys)
    looked_up = {}, bad = 0;
    if (left > 0 && (lane & 31) < 2 * AHEAD) {
      const int page = c.table[(int64_t)q.index * c.table_pitch + (key >> c.page_shift)];
      const int slot = key & ((1 << c.page_shift) - 1);
      if (page >= 0 && page < c.pages) {
        if (is_v) {
          at = (uint64_t)c.v + hk * c.sv.z + page * c.sv.p + slot * c.sv.y - BIAS;
          looked_up = read_scales(c.v_scale + hk * c.svs.z + page * c.svs.p + slot * c.svs.y, c.svs.y, side_by_side, left);
        } else {
          at = (uint64_t)c.k + hk * c.sk.z + page * c.sk.p + slot * c.sk.y - BIAS;
          looked_up = read_scales(c.k_scale + hk * c.sks.z + page * c.sks.p + slot * c.sks.y, c.sks.y, side_by_side, left);
        }
        at |= 1ull << 63;
      } else {
        bad = 0xffff;
      }
    }
    at_lo = (uint32_t)at, at_hi = (uint32_t)(at >> 32);
  };
  // The scales that were looked up, to LDS: of keys that a tile does not have 0, and of those that count as NaN as said above.
  // (Apart from the above, so that the first transfers do not wait for them.)
  auto keep_scales = [&](int i) __attribute__((always_inline)) {
    const int t = i + (lane >> 1 & (AHEAD - 1)), left = row_end - (tile0 + w + WAVES * t) * KEYS - 16 * (lane & 1);
    const bool is_v = lane >= 32;
    uint16_t v[16];
    __builtin_memcpy(v, &looked_up, 32);
#pragma unroll
    for (int e = 0; e < 16; e++) {
      if (e >= left) v[e] = 0;
      if (!scale_fits(bits_to_half(v[e]))) bad |= 1u << e;
    }
    bad |= __shfl_xor((int)bad, 32);
#pragma unroll
    for (int e = 0; e < 16; e++)
      if (bad >> e & 1) v[e] = is_v ? 0 : 0x7e00;
    if ((lane & 31) < 2 * AHEAD) {
      unsigned char* const to = sm + SCALES + ((t & (2 * AHEAD - 1)) * KEYS + 16 * (lane & 1)) * 2;
      Scales s;
      __builtin_memcpy(&s, v, 32);
      u32x4_t* const here = (u32x4_t*)(to + (is_v ? KIND : 0));
      here[0] = s.lo, here[1] = s.hi;
      if (is_v) {
#pragma unroll
        for (int e = 0; e < 16; e++)
          v[e] = half_to_bits((half_t)__builtin_amdgcn_logf(fmaxf(fabsf((float)bits_to_half(v[e])), 0x1p-25f)));
        __builtin_memcpy(&s, v, 32);
        u32x4_t* const logs = (u32x4_t*)(to + 2 * KIND);
        logs[0] = s.lo, logs[1] = s.hi;
      }
    }
  };
  // Keys, or values, of tile i.
  auto fetch = [&](int i, auto is_k) __attribute__((always_inline)) {
    constexpr bool IS_K = decltype(is_k)::value;
    const int stride = IS_K ? k_stride : v_stride;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int l = (IS_K ? 0 : 32) + 2 * (i & (AHEAD - 1)) + h, left = min(row_end - (tile0 + w + WAVES * i) * KEYS - 16 * h, 16);
      const uint32_t lo = __builtin_amdgcn_readlane(at_lo, l), hi = __builtin_amdgcn_readlane(at_hi, l);
      const u32x4_t desc = {lo, hi & 0xffffu, hi >> 31 ? (uint32_t)((left - 1) * stride + d + BIAS) : 0u, 0x00020000u};
      transfer_once<NI / 2>(lds0 + ((IS_K ? 0 : 2) + (i & 1)) * TILE + h * (NI / 2) * 1024, IS_K ? koff : voff[h], desc);
    }
  };
  const std::true_type is_k{};
  const std::false_type is_v{};

  look_up(0);
  asm volatile("" : "+v"(at_lo), "+v"(at_hi));
  if (tiles > 0) fetch(0, is_k), fetch(0, is_v);
  if (tiles > 1) fetch(1, is_k);
  keep_scales(0);
  if (tiles > 1) wait_vm<3 * NI>();
  else if (tiles > 0) wait_vm<2 * NI>();
  else wait_vm<0>();
  half8_t qf[2 * KP];
  float first_sum = 0.0f;
#pragma unroll
  for (int ks = 0; ks < 2 * KP; ks++) {
    qf[ks] = *(const half8_t*)(sm + SCALES - TILE + ks * 1024 + lane * 16);
    if ((ks >> 1) * 64 + g * 16 + (ks & 1) * 8 >= d) qf[ks] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int ks = 0; ks < 2 * KP; ks++) asm volatile("" : "+v"(qf[ks]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (tiles > 1) fetch(1, is_v);
#pragma unroll
  for (int ks = 0; ks < 2 * KP; ks++)
#pragma unroll
    for (int e = 0; e < 8; e++) first_sum += (float)qf[ks][e];
  {
    float x = first_sum, y = x;  // over the four lanes that share a row
    swap_halves(x, y);
    x = x + y, y = x;
    swap_rows(x, y);
    first_sum = -127.5f * WIDENED * (x + y);
    if (!(fabsf(first_sum) < INFINITY)) first_sum = NAN;
  }
  int offK[KP], offV[DB];
#pragma unroll
  for (int kp = 0; kp < KP; kp++) offK[kp] = k_chunk_off<CPR>(frow, kp * 4 + g);
  {
    // Lanes 2 r and 2 r + 1 of each 16 address 16 codes of row r of eight, and lane c gets the eight of column c: rows in the order
    // of a lane's scores.
    const int c = lane & 15, e = c >> 1, r = 4 * g + (e & 3) + 16 * (e >> 2);
#pragma unroll
    for (int db = 0; db < DB; db++) offV[db] = r * ROWB + ((db ^ value_swizzle<CPR>(r)) << 4) + (c & 1) * 8;
  }
  typedef int int2_t __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) int2_t lds_int2_t;

  float4_t o[DB];
  float m_run = NO_SCORE, l_run = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; db++) o[db] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int end = min(end_of_row(a, q, row), row_end) - 4 * g;  // this lane's first key that its row does not see
  // (of the block's first row, which sees the fewest; of a draft, what is in front of it)
  const int common_end = min(row_end, uniform(TREE ? end_of_common(a, q, 0) : end_of_row(a, q, row_of_list(a, block * ROWS))));
  const float c = a.c / WIDENED;  // (scores are times 2^-24)
  float4_t ones = {0.0f, 0.0f, 0.0f, 0.0f};
  half8_t all_ones;
#pragma unroll
  for (int e = 0; e < 8; e++) all_ones[e] = (half_t)1;
  // Tile i; `next`: there is a tile i + 1, `more`: and a tile i + 2, whose keys and values are asked for as soon as the fragments
  // of this one's are in registers.
  auto tile = [&](int i, auto next, auto more) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value, MORE = decltype(more)::value;
    wait_vm<NEXT ? 3 * NI : NI>();  // its keys have landed
    const unsigned char* const cK = sm + (i & 1) * TILE;
    const unsigned char* const cV = sm + (2 + (i & 1)) * TILE;
    u32x4_t kc[2][KP];
    half4_t ks[2], vs[2], log_vs[2];
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
#pragma unroll
      for (int kp = 0; kp < KP; kp++) kc[kb][kp] = *(const u32x4_t*)(cK + offK[kp] + kb * 16 * ROWB);
      const unsigned char* const scales = sm + SCALES + ((i & (2 * AHEAD - 1)) * KEYS + 16 * kb + 4 * g) * 2;
      ks[kb] = *(const half4_t*)scales;
      vs[kb] = *(const half4_t*)(scales + KIND);
      log_vs[kb] = *(const half4_t*)(scales + 2 * KIND);
    }
    float4_t s[2];
#pragma unroll
    for (int kb = 0; kb < 2; kb++) s[kb] = float4_t{first_sum, first_sum, first_sum, first_sum};
#pragma unroll
    for (int kp = 0; kp < KP; kp++)
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
          s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(widened(kc[kb][kp][2 * h], kc[kb][kp][2 * h + 1]), qf[2 * kp + h], s[kb], 0, 0, 0);
    if constexpr (MORE) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const bool looks = ((i + 2) & (AHEAD - 1)) == 0;
      if (looks) {
        look_up(i + 2);
        asm volatile("" : "+v"(at_lo), "+v"(at_hi));
      }
      fetch(i + 2, is_k);
      if (looks) keep_scales(i + 2);
    }
    wait_vm<MORE ? 3 * NI : NEXT ? 2 * NI : 0>();  // and its values
    int2_t vc[DB];
#pragma unroll
    for (int db = 0; db < DB; db++) vc[db] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2_t*)ADR_LDS_PTR(cV + offV[db]));
    if constexpr (MORE) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int db = 0; db < DB; db++) asm volatile("" : "+v"(vc[db]));
      fetch(i + 2, is_v);
    }
    const int key0 = (tile0 + w + WAVES * i) * KEYS;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r++) s[kb][r] = fmaf(s[kb][r], (float)ks[kb][r], 0.0f);  // (one instruction, with the scale as it is)
    if (key0 + KEYS > common_end) {  // keys that some row does not see
      const int left = end - key0;   // of this lane's row from its first one on
      uint32_t seen = ~0u;
      if constexpr (TREE) seen = tree_window(a, q.row0 + row, key0 - (q.keys - q.rows)) >> 4 * g;
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (16 * kb + r >= left || (TREE && !(seen >> (16 * kb + r) & 1))) s[kb][r] = -INFINITY;
    }
    float mx = NO_SCORE;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r++) mx = fmaxf(mx, fmaf(s[kb][r], c, (float)log_vs[kb][r]));
    float x = mx, y = mx;  // over the four lanes that share a row
    swap_halves(x, y);
    x = fmaxf(x, y), y = x;
    swap_rows(x, y);
    const float top = above(fmaxf(x, y));
    if (__builtin_amdgcn_ballot_w64(top > m_run + GROWN_U8) != 0) {
      const float m_new = fmaxf(m_run, top - BELOW), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      ones *= alpha;
#pragma unroll
      for (int db = 0; db < DB; db++) o[db] *= alpha;
    }
    float sum[2] = {0.0f, 0.0f};
    u32x4_t pf, rest;
#pragma unroll
    for (int kb = 0; kb < 2; kb++)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float2_t e, p;  // (and what rounding takes off p, by one instruction: the product once more, less the rounded one)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          e[j] = __builtin_amdgcn_exp2f(fmaf(s[kb][r + j], c, -m_run));
          sum[j] += e[j];
          p[j] = fmaf(e[j], (float)vs[kb][r + j], 0.0f);
        }
        const half2_t h = __builtin_convertvector(p, half2_t);
#pragma unroll
        for (int j = 0; j < 2; j++) p[j] = fmaf(e[j], (float)vs[kb][r + j], -(float)h[j]);
        pf[kb * 2 + r / 2] = __builtin_bit_cast(uint32_t, h);
        rest[kb * 2 + r / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, half2_t));
      }
    l_run += sum[0] + sum[1];
    ones = __builtin_amdgcn_mfma_f32_16x16x32_f16(all_ones, __builtin_bit_cast(half8_t, pf), ones, 0, 0, 0);
    ones = __builtin_amdgcn_mfma_f32_16x16x32_f16(all_ones, __builtin_bit_cast(half8_t, rest), ones, 0, 0, 0);
#pragma unroll
    for (int db = 0; db < DB; db++) {
      const half8_t v = widened((uint32_t)vc[db][0], (uint32_t)vc[db][1]);
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(half8_t, pf), o[db], 0, 0, 0);
      o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(half8_t, rest), o[db], 0, 0, 0);
    }
  };
  const std::true_type yes{};
  const std::false_type no{};
  int i = 0;
  for (; i + 2 < tiles; i++) {
    tile(i, yes, yes);
    if ((i & 15) == 15) {  // (the offset of what is summed so far)
#pragma unroll
      for (int db = 0; db < DB; db++) o[db] -= ones * (127.5f * WIDENED);
      ones = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  if (i + 1 < tiles) tile(i++, yes, no);
  if (i < tiles) tile(i, no, no);

  Args z = arguments();
  // Merge the wavefronts' results: [wavefront][row][HD] sums, and (maximum, sum) of every row.
  wait_vm<0>();
  __syncthreads();
  float* const xo = (float*)smem;
  float2* const xml = (float2*)(smem + WAVES * 16 * PITCH * 4);
  float x = l_run, y = x;
  swap_halves(x, y);
  x = x + y, y = x;
  swap_rows(x, y);
  if (g == 0) xml[w * 16 + frow] = make_float2(m_run, x + y);
#pragma unroll
  for (int db = 0; db < DB; db++)
    *(float4_t*)(xo + (w * 16 + frow) * PITCH + 16 * db + 4 * g) = o[db] * (1.0f / WIDENED) - ones * 127.5f;
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
      round_means(v, sum, l == 0.0f ? 0.0f : 1.0f / l);
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
    const int again = (int)__ballot(is_far(m_all));  // (not stored above)
    for (int r = w; r < rows; r += WAVES)
      if (again >> r & 1) {
        const int lr = block * ROWS + r;
        row_by_wave_u8<TREE>(arguments(), q, lr / z.group, hk * z.group + lr % z.group, lane);
      }
  }
  if (!SHARED || next_place >= stretch1) break;
  __syncthreads();  // (the next block's transfers go where the results are read)
  }
}

// What the matrix-core kernels take: whole chunks of 16 bytes at 16-byte addresses, 16 key rows within the reach of a
// descriptor's 32-bit offsets, rows that do not overlap.
bool chunks(const SequencesArgs& a) {
  const uintptr_t ptrs = (uintptr_t)a.out | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const int64_t strides = (int64_t)a.so_y | a.so_z | a.sq_y | a.sq_z;
  const int64_t codes = a.sk.y | a.sk.z | a.sk.p | a.sv.y | a.sv.z | a.sv.p;
  auto near = [&](int64_t y) { return y >= a.d && y < 1 << 24; };
  return a.d % 16 == 0 && a.d <= 128 && a.so_x == 1 && a.sq_x == 1 && a.sk.x == 1 && a.sv.x == 1 && ptrs % 16 == 0 &&
         strides % 8 == 0 && strides >= 0 && codes % 16 == 0 && codes >= 0 && near(a.sk.y) && near(a.sv.y) &&
         page_shift(a.page_size) >= 0;
}

}  // namespace

SequencesPlan sequences_u8_plan(const SequencesArgs& a, int cus, int64_t avail) {
  const SequencesPlan any = {SequencesPlan::ANY_LAYOUT, 0, 0, 0, 0, 0};
  // (1: any layout; 2 ... 4: few rows, unshared with two or eight wavefronts, shared; 5 ... 8: many; as sequences_plan)
  const int forced = knob(KNOB_SEQUENCES) >= 1 && knob(KNOB_SEQUENCES) <= 8 ? knob(KNOB_SEQUENCES) : 0;
  if (!chunks(a) || forced == 1) return any;
  const int longest_rows = a.longest_rows > 0 ? std::min(a.longest_rows, a.rows) : a.rows;
  const int64_t most_keys = std::min((int64_t)a.table_width * a.page_size, (int64_t)MOST_KEYS);
  const double longest = a.longest > 0 ? std::min<double>(a.longest, most_keys) : most_keys;
  const int sequences = std::min(a.rows, a.sequences), hd = a.d <= 64 ? 64 : 128;
  // Blocks of all key heads, as far as the host can tell (as in sequences_plan), of either kernel.
  auto blocks_of = [&](int rows) {
    const double full = (double)a.rows * a.group / rows, ends = (double)longest_rows * sequences > 4.0 * a.rows ? sequences : sequences / 2.0;
    return a.kv_heads * (sequences <= 1 ? ceil(full) : std::max(full + ends, (double)sequences));
  };
  const bool one_block = (int64_t)longest_rows * a.group <= FEW;
  const double few_blocks = one_block ? a.kv_heads * std::max((double)a.rows * a.group / FEW, (double)sequences) : blocks_of(FEW);
  static const Costs of_64 = {{5.4, 16, 5.0, 0.89, 2.3}, {6.4, 5.0, 2.6, 5.1, 4.2}, {6.9, 1.6, 10, 0.7, 7.4},
                              {6.8, 20, 1.6, 3.4, 6.6}, {7.7, 14, 1.4, 7.2, 9.1}, {9.7, 1.3, 0.013}, {9.9, 1.5, 0.017}, 0.85, 1.4, 0.012};
  static const Costs of_128 = {{6.8, 18, 4.0, 1.7, 3.7}, {7.4, 6.2, 2.7, 6.1, 5.5}, {8.3, 1.7, 11, 1.1, 8.3},
                               {8.6, 26, 3.4, 4.3, 6.5}, {10, 20, 2.7, 8.8, 13}, {12, 0.99, 0.02}, {12, 1.1, 0.025}, 1.4, 2.6, 0.018};
  // Shared few rows: as many workgroups as a unit holds at once, six of heads up to 64 by their 150 registers (three wavefronts to a SIMD), four of
  // 128 by their LDS.  Stretches are equal, and more workgroups are a second round.  us, six and eight of heads of 64: eight sequences
  // of 20000 to 40000 keys (20 / 20) 118, 132; 40 of 500 to 8000 (32 / 4) 29, 35; one of 30000 (12 / 12) 19, 25.  Four and six of 128: eight
  // (40 / 8) 92, 109.
  SequencesPlan p = {SequencesPlan::FEW_ROWS, 2, 0, 0, 1, 0};
  plan_by_cost(p, a, cus, avail, few_blocks, blocks_of(MANY), longest, 8, std::max(1, (hd == 64 ? 6 : 4) * cus / a.kv_heads),
               hd == 64 ? of_64 : of_128);
  if (forced) p.kind = forced <= 4 ? SequencesPlan::FEW_ROWS : SequencesPlan::TILES;
  const bool few = p.kind == SequencesPlan::FEW_ROWS;
  const int rows = few ? FEW : MANY, keys = few ? FEW_KEYS : MANY_KEYS;
  const double full = (double)a.rows * a.group / rows;
  if (forced) {  // (shared in small parts, so that short sequences are divided too)
    const bool divides = forced == 4 || (forced > 6 && a.sequences <= 256 && full + sequences < 1000);
    p.waves = forced == 3 || forced == 6 || forced == 8 ? 8 : forced == 5 || forced == 7 ? 4 : 2;
    p.parts = divides ? std::max(16, cus / a.kv_heads) : 0;
    p.least = 1;
  }
  const double most_tiles = ((double)a.rows * a.group / rows + a.sequences) * (most_keys / keys + 2.0);
  for (p.shift = FEW_SHIFT; most_tiles > ldexp(0x1p29, p.shift) && p.shift < 25; p.shift++) {}
  const int64_t part = ((few ? 2 : 1) * (int64_t)rows * (hd * 4 + 8) + (int64_t)sizeof(Seam)) * a.kv_heads;
  p.parts = (int)std::min<int64_t>(p.parts, avail / part);
  if (p.parts < 2) p.parts = 0;
  if (p.parts == 0 && most_blocks(a, rows) > LAUNCH_BLOCKS) return any;
  p.workspace_bytes = p.parts * part;
  return p;
}

template <int HD, bool TREE>
static hipError_t launch_blocks(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  const bool few = p.kind == SequencesPlan::FEW_ROWS;
  const int rows = few ? FEW : MANY;
  Job job;
  (SequencesArgs&)job = a;
  job.page_shift = page_shift(a.page_size);
  job.parts = p.parts, job.shift = p.shift, job.least = p.least;
  job.per_head = 1.0 / a.group;
  job.longest_first = p.longest_first;
  const int64_t part_rows = (int64_t)(few ? 2 : 1) * p.parts * a.kv_heads * rows;
  job.part_o = (float*)workspace;
  job.part_ml = (float2*)(job.part_o + part_rows * HD);
  job.seams = (Seam*)(job.part_ml + part_rows);
  const int64_t most = most_blocks(a, rows), shared = (int64_t)p.parts * a.kv_heads;
  const int64_t blocks = p.parts == 0 ? most : few ? shared : std::max(shared, most);
  if (blocks > LAUNCH_BLOCKS) return hipErrorInvalidConfiguration;
  const int at_once = std::min(rows, 1024 / HD);  // rows of the joining workgroups
  const dim3 grid((unsigned)blocks), join((unsigned)((few ? p.parts - 1 : p.parts / 2) * a.kv_heads * (rows / at_once)));
  const dim3 threads(64 * p.waves);
  const size_t few_lds = (size_t)p.waves * few_bytes(HD);
  if (few && p.parts > 0) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_u8_few_rows_kernel<HD, 2, true, TREE>), grid, threads, few_lds, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, FEW, true>), join, dim3(256), 0, stream, job);
  } else if (few && p.waves == 8) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_u8_few_rows_kernel<HD, 8, false, TREE>), grid, threads, few_lds, stream, job);
  } else if (few) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_u8_few_rows_kernel<HD, 2, false, TREE>), grid, threads, few_lds, stream, job);
  } else if (p.parts > 0) {
    if (p.waves == 8) hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, true, true, 2, TREE, true>), grid, threads, 0, stream, job);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, true, true, 1, TREE, true>), grid, threads, 0, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, MANY, true>), join, dim3(256), 0, stream, job);
  } else if (p.waves == 8) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, true, false, 2, TREE, true>), grid, threads, 0, stream, job);
  } else {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, true, false, 1, TREE, true>), grid, threads, 0, stream, job);
  }
  return hipGetLastError();
}

hipError_t launch_attention_u8(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  if (p.kind == SequencesPlan::ANY_LAYOUT) {
    const int64_t grid = std::min<int64_t>(((int64_t)a.rows * a.heads + 3) / 4, 1 << 22);
    Job job = {};
    (SequencesArgs&)job = a;
    hipLaunchKernelGGL(attention_u8_any_layout_kernel, dim3((unsigned)grid), dim3(256), 0, stream, job);
    return hipGetLastError();
  }
  if (a.mask == MASK_TREE) return a.d <= 64 ? launch_blocks<64, true>(stream, a, p, workspace) : launch_blocks<128, true>(stream, a, p, workspace);
  return a.d <= 64 ? launch_blocks<64, false>(stream, a, p, workspace) : launch_blocks<128, false>(stream, a, p, workspace);
}

}  // namespace adr
