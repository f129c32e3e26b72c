// The kernel of attention over several sequences for many rows, over values of 16 or of 8 bits.
#pragma once

#include <algorithm>
#include <type_traits>

#include "attention_work.hpp"

namespace adr {
namespace {

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
// rows that the mask hides, compute of a tile is in the time and not in the operations).  HD = 128 keeps 24 to 40 vector registers
// in scratch memory at those beginnings and ends, none in the loop; HD = 64 none.  With trees 37 to 45, 4 to 10 of them in the loop, where a
// row's bits are looked at.
//
// U8: the cache is one of codes (attention_u8.hip, which explains the arithmetic, and why probabilities have 11 bits here and 22 in few
// rows).  They lie in LDS as they come and are widened behind its reads: a wavefront widens all of a tile, 128 instructions, where one that
// widened a quarter for all four would have half of that and the tile's way through LDS once more.  A lane reads 16 codes of a key at once, for
// two steps of the product.  Scales come for four tiles at a time, one for each wavefront, by transfers of their own: the table's entries, the
// scales' words, and what is made of them, each a half tile behind the other.  A piece of 1024 rows over 8025 keys (32 / 8 heads of 128) 163 to
// 170 us = 770 to 740 TFLOP/s, where values in 16 bits take 136 to 146: 425 vector instructions for each of a wavefront's tiles (25100 for 59, starts and
// ends among them), the vector ALU busy 64 % of the time beside matrix cores that are busy 36 %.  HD = 128 keeps 40 to 64 vector registers in
// scratch, none in the loop; with trees 56 to 70, some 40 of them in the loop over two tiles, where bits are looked at; HD = 64 none, or with
// trees and shared keys nine words.
template <int HD, bool PAGED, bool SHARED, int GROUPS, bool TREE = false, bool U8 = false>
__global__ __launch_bounds__(256 * GROUPS, 2) void attention_tiles_kernel(Job) {
  static_assert(PAGED || !U8, "codes are in pages");
  constexpr int BYTES = U8 ? 1 : 2;    // of a value of the tiles
  constexpr int CHUNK = 16 / BYTES, CPR = HD / CHUNK, KEYS = 64, ROWS = 128;
  constexpr int TILE = KEYS * HD * BYTES;  // bytes of one K or V tile
  constexpr int NI = TILE / 1024 / 4;  // transfers per wavefront and tile: 16 rows
  constexpr int DS = HD / 16;          // MFMA k-steps over the head dimension
  constexpr int DT = HD / 32;          // 32-wide output column tiles
  constexpr int ROWB = HD * BYTES;     // bytes per tile row
  constexpr int BIAS = NI * 1024;      // bytes that descriptors start ahead, so that no offset is negative
  // K0 K1 V0 V1 of each group (of codes: room for the queries on their way, and the results)
  constexpr int GROUP_BYTES = !U8 ? 4 * TILE : HD == 128 ? 52 * 1024 : 28 * 1024;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[GROUPS * GROUP_BYTES];
  // U8: what has been asked for of a tile's 64 keys (pages, and words that hold a key's and a value's scale), of each wavefront; and
  // eight tiles' scales as they are used: factors of the scores, scales of the values, and their logarithms
  __shared__ __attribute__((aligned(16))) uint32_t asked[U8 ? 4 * GROUPS : 1][3][KEYS];
  __shared__ __attribute__((aligned(16))) float scales[U8 ? GROUPS : 1][8][3][KEYS];
  __shared__ __attribute__((aligned(16))) float unit_scales[KEYS];
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
  unsigned char* const sm = smem + group * GROUP_BYTES;
  const uint32_t lds0 = (uint32_t)(uintptr_t)ADR_LDS_PTR(smem) + group * GROUP_BYTES;
  const int d = a.d, k_stride = (int)a.sk.y, v_stride = (int)a.sv.y;
  // The queries' fragments, by way of the values' LDS, so that nothing waits for them before the first keys are on their
  // way.  (Chunks behind the head dimension are zeros below.)
  static_assert(4 * DS * 1024 <= GROUP_BYTES - 2 * TILE, "the queries fit the values' tiles");
  auto query_col = [&](int ds) __attribute__((always_inline)) { return U8 ? (ds >> 1) * 32 + g * 16 + (ds & 1) * 8 : ds * 16 + g * 8; };
  const half_t* const qrow = a.q + (int64_t)(hk * a.group + gh) * a.sq_z + (int64_t)(q.row0 + row) * a.sq_y;
#pragma unroll
  for (int ds = 0; ds < DS; ds++) {
    const int col = query_col(ds);
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
    first_edge = uniform(TREE ? end_of_common(a, q, 0) : end_of_row(a, q, row_of_list(a, list0))) / KEYS - tile0;
  }

  // (codes: transposing reads take 16 rows' chunks in pairs, those of 32 lanes rows 4 g ... 4 g + 3 and 8 + 4 g ... 8 + 4 g + 3)
  auto value_swizzle = [](int r) __attribute__((always_inline)) {
    if constexpr (!U8) return v_swz<CPR>(r);
    else return CPR == 8 ? ((r >> 1 & 1) | (r >> 3 & 1) << 1) << 1 : (r >> 3 & 1) << 1;
  };
  // Wavefront w transfers rows 16 w ... 16 w + 15 of a tile, 1 KiB at a time: byte offsets of a lane's chunks in those
  // rows, less the j KiB that the instruction adds; chunks behind the head dimension come as zeros.
  uint32_t koff[NI], voff[NI];
#pragma unroll
  for (int j = 0; j < NI; j++) {
    int krow, kc;
    k_chunk_inv<CPR>(j * 64 + lane, krow, kc);
    const int vrow = (j * 64 + lane) / CPR, vc = (lane % CPR) ^ value_swizzle(vrow);
    const uint32_t ko = (uint32_t)((krow * k_stride + kc * CHUNK) * BYTES + BIAS - j * 1024);
    const uint32_t vo = (uint32_t)((vrow * v_stride + vc * CHUNK) * BYTES + BIAS - j * 1024);
    koff[j] = kc * CHUNK < d ? ko : 0x7fff0000u;
    voff[j] = vc * CHUNK < d ? vo : 0x7fff0000u;
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
    t.bytes = left > 0 ? ((left - 1) * t.stride + d) * BYTES + BIAS : 0;
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
        t.pages = page < 0 ? 0 : (t.base + BYTES * (page * t.page_stride + slot * (int64_t)t.stride)) | 1;
      }
      const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)t.pages, n & 63);
      const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(t.pages >> 32), n & 63);
      t.p = (uint64_t)hi << 32 | (lo & ~1u);
      if (!(lo & 1)) t.bytes = 0;
    }
  };
  const std::true_type is_k{};
  const std::false_type is_v{};
  auto first_tile = [&](const unsigned char* base, int64_t stride, int64_t page_stride, auto k) __attribute__((always_inline)) {
    Next t;
    t.base = (uint64_t)base + (PAGED ? 0 : q.key0 * stride * BYTES) - BIAS;
    t.page_stride = page_stride;
    t.stride = (int)stride;
    t.key = tile0 * KEYS + 16 * w;
    t.pages = 0;
    t.p = t.base + BYTES * (t.key * stride);
    locate(t, k);
    return t;
  };
  Next nk = first_tile((const unsigned char*)a.k + hk * a.sk.z * BYTES, a.sk.y, a.sk.p, is_k);
  Next nv = first_tile((const unsigned char*)a.v + hk * a.sv.z * BYTES, a.sv.y, a.sv.p, is_v);
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
    if constexpr (NI == 1) dma_buffer(dst, decltype(is_k)::value ? koff[0] : voff[0], desc);
    else if constexpr (decltype(is_k)::value) dma_buffer_pair<J>(dst, koff[J], koff[J + 1], desc);
    else dma_buffer_pair<J>(dst, voff[J], voff[J + 1], desc);
  };
  // U8.  Scales of tile t of the group (a lane has a key), in three steps.  Transfers are made in any case, so that the waits count
  // right: of what is not there, some other word.
  uint32_t upper = 0;  // bits: the scale is in its word's upper half
  const float factor = U8 ? a.c / WIDENED : 0.0f;  // of the scores, which are times 2^-24
  auto key_of = [&](int t) __attribute__((always_inline)) { return (tile0 + t) * KEYS + lane; };
  auto page_word = [&](int t) __attribute__((always_inline)) {
    const int key = key_of(t);
    return key < row_end ? a.table + (int64_t)q.index * a.table_pitch + (key >> a.page_shift) : a.row_offsets;
  };
  auto scale_words = [&](int t, int page, const half_t*& k, const half_t*& v) __attribute__((always_inline)) {
    const int key = key_of(t), slot = key & ((1 << a.page_shift) - 1);
    k = v = (const half_t*)a.row_offsets;
    if (key < row_end && page >= 0 && page < a.pages) {
      k = a.k_scale + hk * a.sks.z + page * a.sks.p + slot * a.sks.y;
      v = a.v_scale + hk * a.svs.z + page * a.svs.p + slot * a.svs.y;
    }
  };
  // As they are used: of keys that are not there whatever is finite, of those that count as NaN a factor of NaN and values of 0.
  // (A factor of 0 is the smallest number instead: hidden scores stay -inf.)
  auto keep = [&](int t, int page, half_t ks, half_t vs) __attribute__((always_inline)) {
    const bool there = key_of(t) < row_end, good = page >= 0 && page < a.pages && scale_fits(ks) && scale_fits(vs);
    const float k = !there ? 1.0f : !good ? NAN : (float)ks == 0.0f ? 0x1p-126f : (float)ks * factor;
    const float v = there && good ? (float)vs : 0.0f;
    float(*const to)[KEYS] = scales[U8 ? group : 0][t & 7];
    to[0][lane] = k, to[1][lane] = v, to[2][lane] = __builtin_amdgcn_logf(fmaxf(fabsf(v), 0x1p-25f));
  };
  const uint32_t asked_lds = (uint32_t)(uintptr_t)ADR_LDS_PTR(&asked[U8 ? 4 * group + w : 0][0][0]);
  auto whole_word = [](const void* p) __attribute__((always_inline)) { return (const void*)((uintptr_t)p & ~(uintptr_t)3); };
  // In the second half of tile i; what is asked for there has landed at the end of the first half of tile i + 1.
  auto scales_step = [&](int i) __attribute__((always_inline)) {
    if constexpr (U8) {
      if ((i & 3) == 0) {
        dma_global_word(asked_lds, page_word(i + 4 + w));
      } else if ((i & 3) == 1) {
        const half_t *k, *v;
        scale_words(i + 3 + w, (int)asked[4 * group + w][0][lane], k, v);
        upper = ((uintptr_t)k >> 1 & 1) | ((uintptr_t)v & 2);
        dma_global_word(asked_lds + KEYS * 4, whole_word(k));
        dma_global_word(asked_lds + 2 * KEYS * 4, whole_word(v));
      } else if ((i & 3) == 2) {
        const uint32_t* const words = &asked[4 * group + w][0][lane];
        const uint32_t k = words[KEYS], v = words[2 * KEYS];
        keep(i + 2 + w, (int)words[0], bits_to_half((uint16_t)(upper & 1 ? k >> 16 : k)), bits_to_half((uint16_t)(upper & 2 ? v >> 16 : v)));
      }
    }
  };
  const std::integral_constant<int, 0> pair0{};
  const std::integral_constant<int, NI < 4 ? 0 : NI / 2 - 1> pair1{};  // (the last pair, where there are two)
  auto tile_transfers = [&](Next& t, auto k, int buf) __attribute__((always_inline)) {
    transfer(t, k, buf, pair0);
    if constexpr (NI > 2) transfer(t, k, buf, pair1);
    advance(t, k);
  };
  // What is waited for at the end of each half: all transfers but those issued in it, of values, or of keys, and of scales.
  auto wait_landed = [&](auto k, int i) __attribute__((always_inline)) {
    if (U8 && decltype(k)::value && (i & 3) == 0) wait_vm<NI + 1>();
    else if (U8 && decltype(k)::value && (i & 3) == 1) wait_vm<NI + 2>();
    else wait_vm<NI>();
    if (U8 && decltype(k)::value && (i & 3) == 2) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (scales are there for the others)
  };

  tile_transfers(nk, is_k, 0);
  tile_transfers(nk, is_k, 1);
  if constexpr (U8) {  // the first four tiles' scales, one to each wavefront
    const half_t *k, *v;
    const int page = *page_word(w);
    scale_words(w, page, k, v);
    keep(w, page, *k, *v);
    unit_scales[lane] = 1.0f;  // (each wavefront: nobody waits for another's)
  }
  // LDS fragment offsets.  K: lane -> tile row frow (+32), chunk 2*ds + g.
  int offK[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ds++) offK[ds] = k_chunk_off<CPR>(frow, U8 ? (ds >> 1) * 2 + g : ds * 2 + g);
  wait_vm<NI>();  // the queries and the first K tile have landed
  half8_t qf[DS];  // (operand B of S^T = K Q^T: lane -> row frow, head-dimension group g)
#pragma unroll
  for (int ds = 0; ds < DS; ds++) {
    qf[ds] = *(const half8_t*)(sm + 2 * TILE + (w * DS + ds) * 1024 + lane * 16);
    if (query_col(ds) >= d) qf[ds] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
  }
#pragma unroll
  for (int ds = 0; ds < DS; ds++) asm volatile("" : "+v"(qf[ds]));
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (values come there behind the next barrier)
  float first_sum = 0.0f;  // of the scores
  if constexpr (U8) {
#pragma unroll
    for (int ds = 0; ds < DS; ds++)
#pragma unroll
      for (int e = 0; e < 8; e++) first_sum += (float)qf[ds][e];
    first_sum = -127.5f * WIDENED * pair_sum(first_sum);
    if (!(fabsf(first_sum) < INFINITY)) first_sum = NAN;
  }
  // V (transposing read): in each group of 16 lanes, lanes 4r..4r+3 address 16 consecutive halves of tile row r, and
  // lane i of the group receives column i of that 4 x 16 block.  Group b = (lane / 16) % 2 takes columns 16b.. of the
  // 32-column tile, g the rows 4g..4g+3.
  int offV[DT];
  {
    // (codes: lanes 2 e and 2 e + 1 address 16 of row 4 g + e, and from the fifth on 4 further, and lane i receives the eight of
    // column i)
    const int s = lane & 15, b = (lane >> 4) & 1, r = U8 ? (s >> 1 & 3) + 8 * (s >> 3) : s >> 2;
    const int row = 4 * g + r;  // + 32*kt + 16*t + 8*h, all multiples of 8: row & 3 == r & 3
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
      const int chunk = U8 ? 2 * dt + b : 4 * dt + 2 * b + ((s & 3) >> 1);
      offV[dt] = row * ROWB + ((chunk ^ value_swizzle(row)) << 4) + (s & 1) * 8;
    }
  }

  float16_t o[DT], sa[2], sb[2];  // sums of P.V; scores of two tiles in turn
  float sum_of_p = 0.0f;          // U8: of the rounded probabilities, in this lane
  const float* by = unit_scales;  // U8: factors of the scores of the tile whose probabilities come next
  constexpr float MOST = U8 ? GROWN_U8 : GROWN;
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
  u32x4_t kc[NG][2];  // U8: the codes of two steps, of each 32 keys
  typedef int int2_t __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) int2_t lds_int2_t;
  int2_t vc[NG][4];

  auto read_k = [&](const unsigned char* cK, int c) __attribute__((always_inline)) {
    if constexpr (U8) {
#pragma unroll
      for (int j = 0; j < 2; j++) kc[c][j] = *(const u32x4_t*)(cK + offK[2 * c] + j * 32 * ROWB);
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) kf[c][j] = *(const half8_t*)(cK + offK[2 * c + (j >> 1)] + (j & 1) * 32 * ROWB);
    }
  };
  auto key_operand = [&](int c, int f) __attribute__((always_inline)) {
    if constexpr (U8) return widened(kc[c][f & 1][2 * (f >> 1)], kc[c][f & 1][2 * (f >> 1) + 1]);
    else return kf[c][f];
  };
  auto value_operand = [&](int c, int f) __attribute__((always_inline)) {
    if constexpr (U8) return widened((uint32_t)vc[c][f][0], (uint32_t)vc[c][f][1]);
    else return vf[c][f];
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
      if constexpr (U8) {
        vc[c][j] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_int2_t*)ADR_LDS_PTR(p0));
        continue;
      }
      const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0));
      const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)ADR_LDS_PTR(p0 + 8 * ROWB));
      vf[c][j] = __builtin_shufflevector(__builtin_bit_cast(half4_t, lo), __builtin_bit_cast(half4_t, hi),
                                         0, 1, 2, 3, 4, 5, 6, 7);
    }
  };

  // First half of tile i: the scores of tile i + 1 on the matrix cores (K buffer KB), and the
  // probabilities of tile i on the vector ALU.
  auto half1 = [&](int i, auto do_s, auto do_p, auto do_pv, auto kbuf, float16_t (&cur)[2], float16_t (&nxt)[2])
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
    float4_t ks[2], vs[2];  // U8: the tile's factors and scales, of four keys and the next four
    auto read_scales = [&](int x) __attribute__((always_inline)) {
      if constexpr (U8 && P) {
        const int key = 32 * (x >> 2) + 8 * (x & 3) + 4 * g;
        if (x < 8) ks[x & 1] = *(const float4_t*)(by + key), vs[x & 1] = *(const float4_t*)&scales[group][i & 7][1][key];
      }
    };
    read_scales(0);
    read_scales(1);
    auto stage_exponent = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e++) ex[e] = fmaf(cur[k * VP >> 4][(k * VP & 15) + e], U8 ? ks[k * VP >> 2 & 1][(k * VP & 3) + e] : a.c, -m_run);
    };
    auto stage_power = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e++) pw[e] = __builtin_amdgcn_exp2f(ex[e]);
    };
    auto stage_round = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < VP; e += 2) {
        const int x = k * VP + e;
        float2_t e2 = {pw[e], pw[e + 1]};
        if constexpr (U8) e2 = float2_t{pw[e] * vs[x >> 2 & 1][x & 3], pw[e + 1] * vs[x >> 2 & 1][(x & 3) + 1]};
        uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(e2, half2_t));
        sum[0] += pw[e];
        sum[1] += pw[e + 1];
        asm volatile("" : "+v"(bits), "+v"(sum[0]), "+v"(sum[1]));
        pf[x >> 4][x >> 3 & 1][(x & 7) / 2] = bits;
        if constexpr (U8) {
          sum_of_p = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, bits), half2_t{(half_t)1, (half_t)1}, sum_of_p, false);
          if ((x & 3) == 2) read_scales((x >> 2) + 2);
        }
      }
    };
    if constexpr (HD == 128) __builtin_amdgcn_s_setprio(1);
    if constexpr (P) stage_exponent(0);
    if constexpr (S) {
#pragma unroll
      for (int kt = 0; kt < 2; kt++)
#pragma unroll
        for (int r = 0; r < 16; r++) nxt[kt][r] = U8 ? first_sum : 0.0f;
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
          nxt[f & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key_operand(c, f), qf[2 * c + (f >> 1)], nxt[f & 1], 0, 0, 0);
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
    wait_landed(is_v, i);
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
    scales_step(i);
    // U8: the factors of the next tile's scores, and its values' logarithms, of four keys and the next four.  Where some keys are not
    // seen, scores are multiplied before those are taken out, and by ones from then on.
    const float(*const next_scales)[KEYS] = scales[U8 ? group : 0][(i + 1) & 7];
    if constexpr (U8 && MAX) by = next_scales[0];
    float4_t ks[2], logs[2];
    auto read_scales = [&](int x) __attribute__((always_inline)) {
      if constexpr (U8 && MAX) {
        const int key = 32 * (x >> 2) + 8 * (x & 3) + 4 * g;
        if (x < 8) ks[x & 1] = *(const float4_t*)(by + key), logs[x & 1] = *(const float4_t*)(next_scales[2] + key);
      }
    };
    if constexpr (MAX) {
      if (i + 1 >= first_edge) {
        // this lane's first masked key, counted from its own first one
        int end = lane_end - (tile0 + i + 1) * KEYS - 4 * g;
        if constexpr (U8) {
#pragma unroll
          for (int x = 0; x < 8; x++) {
            const float4_t f = *(const float4_t*)(by + 32 * (x >> 2) + 8 * (x & 3) + 4 * g);
#pragma unroll
            for (int e = 0; e < 4; e++) nxt[x >> 2][4 * (x & 3) + e] *= f[e];
          }
          by = unit_scales;
        }
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
          for (int r = 0; r < 16; r++) {
            asm volatile("" : "+v"(end));  // (one comparison at a time: 32 would take as many scalar register pairs)
            if (32 * kt + 8 * (r >> 2) + (r & 3) >= end) nxt[kt][r] = -INFINITY;
          }
        if constexpr (TREE) {
#pragma unroll
          for (int kt = 0; kt < 2; kt++) {
            uint32_t seen = tree_window(a, q.row0 + row, (tile0 + i + 1) * KEYS + 32 * kt - (q.keys - q.rows)) >> 4 * g;
#pragma unroll
            for (int r = 0; r < 16; r++) {
              asm volatile("" : "+v"(seen));
              if (!(seen >> (8 * (r >> 2) + (r & 3)) & 1)) nxt[kt][r] = -INFINITY;
            }
          }
        }
      }
    }
    read_scales(0);
    read_scales(1);
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
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value_operand(c, f), __builtin_bit_cast(half8_t, pf[kt][t]), o[dt], 0, 0, 0);
        }
        if constexpr (MAX) {
          const int first = (4 * c + j - FIRST) * PER * 2;
          if (first >= 0 && first < 32) {
#pragma unroll
            for (int e = 0; e < PER; e++) {
              const int x = first + 2 * e;
              float s0 = nxt[x >> 4][x & 15], s1 = nxt[x >> 4][(x & 15) + 1];
              if constexpr (U8) {
                s0 = fmaf(s0, ks[x >> 2 & 1][x & 3], logs[x >> 2 & 1][x & 3]);
                s1 = fmaf(s1, ks[x >> 2 & 1][(x & 3) + 1], logs[x >> 2 & 1][(x & 3) + 1]);
                if ((x & 3) == 2) read_scales((x >> 2) + 2);
              }
              mx2[e & 1] = fmaxf(fmaxf(mx2[e & 1], s0), s1);
            }
          }
          if (first == 32) mx = above(pair_max(fmaxf(mx2[0], mx2[1])) * (U8 ? 1.0f : a.c));  // in log2 units (c > 0)
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (MAX) {
      // (codes, every 16th tile as well: the offset of what is summed so far is taken off it, as attention_u8.hip says)
      if (__builtin_amdgcn_ballot_w64(mx > m_run + MOST) != 0 || (U8 && (i & 15) == 15)) {
        const float m_new = fmaxf(m_run, mx - BELOW);
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
        float offset = 0.0f;
        if constexpr (U8) offset = pair_sum(sum_of_p) * (127.5f * WIDENED) * alpha, sum_of_p = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
          for (int r = 0; r < 16; r++) o[dt][r] = U8 ? fmaf(o[dt][r], alpha, -offset) : o[dt][r] * alpha;
      }
    }
    advance(nk, is_k);
    wait_landed(is_k, i);
    barrier();
  };
  auto idle = [&](int i) __attribute__((always_inline)) {
    tile_transfers(nv, is_v, 2 + ((i + 1) & 1));
    wait_landed(is_v, i);
    barrier();
    scales_step(i);
    tile_transfers(nk, is_k, (i + 1) & 1);
    wait_landed(is_k, i);
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
    half1(-1, yes, no, no, even, sb, sa);
    half2(-1, no, yes, yes, odd, sa);
    for (i = 0; i + 2 < active; i += 2) {
      half1(i, yes, yes, yes, odd, sa, sb);
      half2(i, yes, yes, yes, even, sb);
      half1(i + 1, yes, yes, yes, even, sb, sa);
      half2(i + 1, yes, yes, yes, odd, sa);
    }
    if (i + 1 < active) {
      half1(i, yes, yes, yes, odd, sa, sb);
      half2(i, yes, yes, no, even, sb);
      half1(i + 1, no, yes, yes, even, sb, sa);
      half2(i + 1, yes, no, no, odd, sa);
    } else {
      half1(i, no, yes, yes, odd, sa, sb);
      half2(i, yes, no, no, even, sb);
    }
    i = active;
  }
  for (; i < steps; i++) idle(i);  // tiles this wavefront has no part in
  wait_vm<0>();  // (transfers of no bytes write zeros)
  if constexpr (U8) {
    const float offset = pair_sum(sum_of_p) * 127.5f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[dt][r] = fmaf(o[dt][r], 1.0f / WIDENED, -offset);
  } else if constexpr (PAGED) {
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
    float4_t* const theirs = (float4_t*)(smem + (1 - group) * GROUP_BYTES) + at;
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
  if constexpr (PAGED && !U8) {
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
    constexpr int PITCH = HD * 2 / GROUPS + 16, CHUNKS = HD / 8 / GROUPS;
    static_assert(EXCHANGE + 4 * 32 * PITCH <= GROUP_BYTES, "the output's slots fit the LDS");
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
      if (!U8 && bad && (TREE || (q.rows > 1 && z.mask == ADR_MASK_CAUSAL)) &&
          hidden_reaches(z, q, hk, TREE ? end_of_common(z, q, 0) : end_of_row(z, q, row_of_list(z, list0 + min(__builtin_ctz(bad), wave_rows - 1))),
                         end_of_row(z, q, row_of_list(z, block * ROWS + rows - 1)), lane))
        again |= bad;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (behind the stores above)
      for (int r = 0; r < wave_rows; r++)
        if (again >> r & 1) {
          if constexpr (U8) row_by_wave_u8<TREE>(arguments(), q, (list0 + r) / z.group, hk * z.group + (list0 + r) % z.group, lane, col0, col0 + 32 * MINE);
          else row_by_wave<TREE>(arguments(), q, (list0 + r) / z.group, hk * z.group + (list0 + r) % z.group, lane, col0, col0 + 32 * MINE);
        }
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

// ---- the choice, on the host ------------------------------------------------------------------------------------

int page_shift(int page_size) { return page_size >= 16 && (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1; }

// Blocks of all key heads that there can be, and as many as a launch of 256 threads to each may have.
int64_t most_blocks(const SequencesArgs& a, int rows) {
  return ((int64_t)a.rows * a.group / rows + std::min(a.rows, a.sequences)) * a.kv_heads;
}
constexpr int64_t LAUNCH_BLOCKS = 0x7fffffff / 256;

// Of the ways to share many rows' keys the one that should take least, of a kernel whose tiles take `one` us with a compute unit to
// itself and `two` for two beside each other, and `way` for a part's way through memory.
inline void plan_tiles(SequencesPlan& p, const SequencesArgs& a, int cus, double blocks, double longest, double one, double two,
                       double way) {
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

// Of all forms the one that should take least, for calls that may go through either kernel whatever their rows are: few rows with two
// wavefronts to a block, with `waves`, or shared; many rows with four or eight, or shared.
//
// us, with `keys` thousands of keys of the longest sequence and `blocks` for each compute unit: a block by itself takes start + alone *
// keys, all of them `all` + (block + read * keys) * blocks, and the longer of the two counts, or a little more than either where they
// are level.  Shared many rows as in plan_tiles.  Fitted to the times of every form over 36800 drawn batches (1 to 1024 rows and sequences,
// 1 to 65000 keys, 12 to 40 heads of 64 to 128 in 1 to 32 key heads): over others, the form that is taken needs 1.03 times the time of the
// best, all together; one in a hundred 1.3 times.  (By rows alone, as for attention_paged_f16, 1.15 and 1.9.)
struct Cost {
  double start, alone, all, block, read;
  double us(double keys, double blocks) const {
    const double x = start + alone * keys, y = all + (block + read * keys) * blocks;
    return sqrt(sqrt(x * x * x * x + y * y * y * y));
  }
};
struct SharedCost {
  double start, tile, part;
};
struct Costs {
  Cost two, waves, few_shared, four, eight;
  SharedCost four_shared, eight_shared;
  double tile, tiles, way;  // as in plan_tiles, for the number of parts
};

inline void plan_by_cost(SequencesPlan& p, const SequencesArgs& a, int cus, int64_t avail, double few_blocks, double many_blocks, double longest,
                         int waves, int few_parts, const Costs& c) {
  const double keys = longest / 1000, few = few_blocks / cus, many = many_blocks / cus;
  double best = HUGE_VAL;
  auto take = [&](double us, SequencesPlan::Kind kind, int with, int parts, int least) {
    if (us < best) best = us, p.kind = kind, p.waves = with, p.parts = parts, p.least = least;
  };
  const int hd = a.d <= 64 ? 64 : 128;
  auto fits = [&](int64_t slots) { return avail / ((slots * (hd * 4 + 8) + (int64_t)sizeof(Seam)) * a.kv_heads) >= 2; };
  p.longest_first = a.sequences > 1 && few > 1.0;
  take(c.two.us(keys, few), SequencesPlan::FEW_ROWS, 2, 0, 1);
  take(c.waves.us(keys, few), SequencesPlan::FEW_ROWS, waves, 0, 1);
  if (a.sequences <= 256 && few_parts > 1 && fits(2 * FEW)) take(c.few_shared.us(keys, few), SequencesPlan::FEW_ROWS, 2, few_parts, 1);
  if ((int64_t)(a.longest_rows > 0 ? std::min(a.longest_rows, a.rows) : a.rows) * a.group <= FEW) return;  // (a block for each sequence)
  take(c.four.us(keys, many), SequencesPlan::TILES, 4, 0, 4);
  take(c.eight.us(keys, many), SequencesPlan::TILES, 8, 0, 4);
  if (a.sequences > 256 || !fits(MANY)) return;
  const bool single = a.sequences == 1;
  const double work = many_blocks * (longest / MANY_KEYS + 1) * (single ? 1.0 : 0.75);
  auto shared = [&](int with, double most, double tile, const SharedCost& cost) {
    double n = std::min(most, sqrt(work * tile / c.way));
    if (single) n = floor(n / many_blocks) * many_blocks;
    if (n < (single ? 2.0 : 1.5) * many_blocks) return;
    take(cost.start + cost.tile * work * tile / (single ? n : n - many_blocks / 2) + cost.part * n, SequencesPlan::TILES, with,
         (int)(n / a.kv_heads + 0.5), 4);
  };
  shared(4, cus * 15 / 16.0, c.tile, c.four_shared);
  shared(4, 2.0 * cus, c.tiles, c.four_shared);
  shared(8, cus, c.tiles / 2, c.eight_shared);
}

}  // namespace
}  // namespace adr
