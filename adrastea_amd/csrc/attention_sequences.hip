// Attention of packed rows of several sequences, over the pages of a cache or over packed keys.
//
//   out[h, row] = sum_x softmax_x( scale <q[h, row], k[x]> / temp ) v[x],   x <= j + n - r under the mask
//
// for row j of a sequence of r rows and n keys.  Query heads come in groups that share a key and value head.

#include <algorithm>
#include <type_traits>

#include "attention_tiles.hpp"


namespace adr {
namespace {

__global__ __launch_bounds__(256) void attention_any_layout_kernel(Job) { rows_one_by_one<false>(arguments()); }

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
//
// TREE: the rows are drafted tokens.  What they see of each other is looked at in the tiles that hold some of them only.
template <int HD, bool PAGED, int WAVES, bool SHARED, bool TREE = false>
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
  Roster<ROWS, KEYS, PAGED, SHARED, TREE && !SHARED> roster;
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
        if constexpr (!TREE) mx = fmaxf(mx, s[kb][r]);
      }
    if constexpr (TREE) {
      const int drafted = (tile0 + w + WAVES * i) * KEYS - (q.keys - q.rows);  // of the tile's first key
      if (drafted > -KEYS) {
        const uint32_t seen = tree_window(a, q.row0 + row, drafted) >> 4 * g;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (!(seen >> (16 * kb + r) & 1)) s[kb][r] = -INFINITY;
      }
#pragma unroll
      for (int kb = 0; kb < 2; kb++)
#pragma unroll
        for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[kb][r]);
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
    if (TREE || (q.rows > 1 && z.mask == ADR_MASK_CAUSAL)) {
      __syncthreads();
      const int bad = uniform(*bad_rows);
      if (bad && hidden_reaches(z, q, hk, end_of_common(z, q, row_of_list(z, block * ROWS + __builtin_ctz(bad))),
                                end_of_row(z, q, row_of_list(z, block * ROWS + rows - 1)), lane))
        again |= bad;
    }
    for (int r = w; r < rows; r += WAVES)
      if (again >> r & 1) {
        const int lr = block * ROWS + r;
        row_by_wave<TREE>(arguments(), q, lr / z.group, hk * z.group + lr % z.group, lane);
      }
  }
  if (!SHARED || next_place >= stretch1) break;
  __syncthreads();  // (the next block's transfers go where the results are read)
  }
}

}  // namespace

// ---- the choice ---------------------------------------------------------------------------------------------

namespace {

// What the matrix-core kernels take: whole chunks of 16 bytes at 16-byte addresses, 16 key rows within the reach of a
// descriptor's 32-bit offsets, rows that do not overlap (a row behind the last key is told by its offset).
bool chunks(const SequencesArgs& a) {
  const uintptr_t ptrs = (uintptr_t)a.out | (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const int64_t strides = (int64_t)a.so_y | a.so_z | a.sq_y | a.sq_z | a.sk.y | a.sk.z | a.sk.p | a.sv.y | a.sv.z | a.sv.p;
  auto near = [&](int64_t y) { return y >= a.d && y < 1 << 24; };
  return a.d % 8 == 0 && a.d <= 128 && a.so_x == 1 && a.sq_x == 1 && a.sk.x == 1 && a.sv.x == 1 && ptrs % 16 == 0 &&
         strides % 8 == 0 && strides >= 0 && near(a.sk.y) && near(a.sv.y) && (!a.table || page_shift(a.page_size) >= 0);
}


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
  bool few = p.kind == SequencesPlan::FEW_ROWS;
  int rows = few ? FEW : MANY, keys = few ? FEW_KEYS : MANY_KEYS;
  const int hd = a.d <= 64 ? 64 : 128;
  const int64_t most_keys = a.table ? std::min((int64_t)a.table_width * a.page_size, (int64_t)MOST_KEYS) : a.keys;
  const double longest = a.longest > 0 ? std::min<double>(a.longest, most_keys) : most_keys;
  // Blocks of all key heads, as far as the host can tell: a sequence's last one is full by half, but where one sequence has
  // most of the rows, the others' only ones.
  const int sequences = std::min(a.rows, a.sequences);
  const double full = (double)a.rows * a.group / rows, ends = (double)longest_rows * sequences > 4.0 * a.rows ? sequences : sequences / 2.0;
  const double blocks = a.kv_heads * (few ? std::max(full, (double)sequences) : sequences <= 1 ? ceil(full) : std::max(full + ends, (double)sequences));
  p.least = 1;
  if (a.mask == MASK_TREE && !forced) {
    // Drafts are often more than a block of few rows, and seldom one of many: either kernel, by what it takes.
    static const Costs of_64 = {{5.6, 9.2, 1.2, 1.2, 5.9}, {5.6, 4.8, 1.2, 2.1, 5.4}, {6.1, 1.2, 8.2, 0.64, 8.1},
                                {6.8, 11, 2.2, 2.9, 8.7}, {7.6, 8.6, 1.3, 6.8, 11}, {9.1, 1.1, 0.015}, {9.9, 1.2, 0.022}, 0.67, 1.02, 0.012};
    static const Costs of_128 = {{5.8, 11, 2.7, 2.3, 9.7}, {5.7, 7.3, 1.9, 4.5, 8.4}, {4.6, 1.5, 8.9, 1.7, 14},
                                 {8.7, 16, 4.8, 3.9, 15}, {10, 12, 4.1, 8.9, 16}, {12, 1.1, 0.016}, {12, 1.0, 0.025}, 1.1, 2.0, 0.018};
    auto blocks_of = [&](int rows) {
      const double full = (double)a.rows * a.group / rows;
      return a.kv_heads * (rows == FEW && (int64_t)longest_rows * a.group <= FEW ? std::max(full, (double)sequences)
                           : sequences <= 1                                      ? ceil(full)
                                                                                 : std::max(full + ends, (double)sequences));
    };
    const double few_blocks = blocks_of(FEW);
    const int each = (hd == 64 ? 2 : 1) * (few_blocks >= 4.0 * cus ? 2 : 1);
    plan_by_cost(p, a, cus, avail, few_blocks, blocks_of(MANY), longest, 4, std::max(1, each * cus / a.kv_heads), hd == 64 ? of_64 : of_128);
    few = p.kind == SequencesPlan::FEW_ROWS;
    rows = few ? FEW : MANY, keys = few ? FEW_KEYS : MANY_KEYS;
  } else if (few) {
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
    plan_tiles(p, a, cus, blocks, longest, one, two, way);
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

template <int HD, bool PAGED, bool TREE = false>
static hipError_t launch_blocks(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  const bool few = p.kind == SequencesPlan::FEW_ROWS;
  const int rows = few ? FEW : MANY;
  Job job;
  (SequencesArgs&)job = a;
  job.page_shift = PAGED ? page_shift(a.page_size) : 0;
  job.parts = p.parts, job.shift = p.shift, job.least = p.least;
  job.part_o = (float*)workspace;
  job.per_head = 1.0 / a.group;
  job.longest_first = p.longest_first;
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
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 2, true, TREE>), grid, threads, few_lds, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, FEW>), join, dim3(256), 0, stream, job);
  } else if (few && p.waves == 2) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 2, false, TREE>), grid, threads, few_lds, stream, job);
  } else if (few) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_few_rows_kernel<HD, PAGED, 4, false, TREE>), grid, threads, few_lds, stream, job);
  } else if (p.parts > 0) {
    if (p.waves == 8) hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, true, 2, TREE>), grid, threads, 0, stream, job);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, true, 1, TREE>), grid, threads, 0, stream, job);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_join_kernel<HD, MANY>), join, dim3(256), 0, stream, job);
  } else if (p.waves == 8) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, false, 2, TREE>), grid, threads, 0, stream, job);
  } else {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attention_tiles_kernel<HD, PAGED, false, 1, TREE>), grid, threads, 0, stream, job);
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
  if (a.mask == MASK_TREE) return a.d <= 64 ? launch_blocks<64, true, true>(stream, a, p, workspace) : launch_blocks<128, true, true>(stream, a, p, workspace);
  if (a.d <= 64) return a.table ? launch_blocks<64, true>(stream, a, p, workspace) : launch_blocks<64, false>(stream, a, p, workspace);
  return a.table ? launch_blocks<128, true>(stream, a, p, workspace) : launch_blocks<128, false>(stream, a, p, workspace);
}

}  // namespace adr
