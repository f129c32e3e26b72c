// Rotary positions, and a step's new keys and values into the pages of the cache.
//
//   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),   t = 2 pi * position * turns[i]
//
// The angle is made where it is used: a table of cosines would be read from memory for every row and has an
// end.  position * turns[i] is a 64-bit product (positions of seven digits leave 2^-33 of a turn), its whole
// turns are taken off in 64 bits, and what is left, at most half a turn, goes through the 32-bit sincospi.
// Each is computed once per row and pair, by a thread of its own, and shared by all heads through LDS.
#include <algorithm>
#include <type_traits>

#include "sequences.hpp"

namespace adr {
namespace {

constexpr int MAX_ROWS = 16;  // of a workgroup

struct RowPlace {   // of one row of the workgroup
  int row;          // -1: none
  int position;
  int64_t k, v;     // element offset of its slot in the cache (head 0); -1: not written
};

struct RotaryJob : RotaryArgs {
  int rows_per_wg;
  int items;  // of a head
};

// The job, read from the kernel's arguments (of which it is the only one) where it is used.  Loads do not move across this:
// kept in registers from the start, all of it would not fit the scalar ones.
typedef const __attribute__((address_space(4))) RotaryJob& Args;
__device__ __forceinline__ Args arguments() {
  auto p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const __attribute__((address_space(4))) RotaryJob*)p;
}

// Queries, keys and values are one list of heads, and each head the same list of items.  VEC: 16 bytes at a time --
// an item is a pair of chunks of 8 values (halves), a chunk of 4 pairs (pairs), or a chunk that passes.  Otherwise it is one
// pair or one value that passes, at any stride.  Values have the same items, with nothing turned.
//
// Bound by memory, and before that by what it takes to find an item: so a thread has the same item of all the heads
// that it goes through, and from head to head only the addresses change.  Items asked for ahead cost registers that
// are wavefronts (us with four ahead, two, none: 4099 rows of 40 heads of 128, pairs, half of the head 21.4, 19.7, 17.4), and
// nobody waits for the stores at the end (17.3 -> 16.4).  15.3 to 17.0 us = 4.9 to 5.5 TB/s; four prompts of 700 to 2500 rows into
// the cache (32 / 8 heads of 128) 39.3 us = 4.4 TB/s.  Nontemporal stores would take 15.1 and 31.6, but what is written here is
// what the attention behind it reads: both together four prompts of 2000 rows 191.2 us, with them 195.4, eight heads of their own
// 80.0 and 84.8.  CACHE false: queries only.
template <bool VEC, bool CACHE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryJob) {
  Args a = arguments();
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  RowPlace* const place = (RowPlace*)smem;                                     // [rows_per_wg]
  float2* const turn = (float2*)(smem + MAX_ROWS * sizeof(RowPlace));          // [rows_per_wg][dims / 2]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int R = a.rows_per_wg, half = a.dims >> 1, items = a.items;
  typedef typename std::conditional<VEC, half8_t, half_t>::type chunk_t;

  const int q_heads = a.q ? a.heads : 0, kv_heads = CACHE ? a.kv_heads : 0, heads = q_heads + 2 * kv_heads;
  const int side_by_side = items < 256 ? 256 / items : 1;  // heads at once
  const int first = items < 256 ? tid / items : 0;
  const int item0 = first < side_by_side ? tid - first * items : items;  // (threads left over have none)
  chunk_t v = {}, v2 = {};

  // Item `in` of a head: its chunks' first values, whether there are two, whether they are turned (but for values).
  struct Item {
    int in, x, x2;
    bool pair, two;
  };
  auto item_at = [&](int in) __attribute__((always_inline)) {
    constexpr int W = VEC ? 8 : 1;  // values of a chunk
    const int count = VEC && !a.pairs ? half >> 3 : VEC ? a.dims >> 3 : half;
    Item t;
    t.in = in;
    t.pair = in < count;
    t.two = t.pair && !(VEC && a.pairs);
    t.x = !t.pair ? (in - count) * W + a.dims : !VEC && a.pairs ? 2 * in : in * W;
    t.x2 = t.x + (a.pairs ? 1 : half);
    return t;
  };
  auto read = [&](const Item& t, int64_t row, int h) __attribute__((always_inline)) {
    const int k = CACHE ? h - q_heads : -1, w = CACHE ? k - kv_heads : -1;
    const half_t* const base = k < 0 ? a.q : w < 0 ? a.k : a.v;
    const int z = k < 0 ? a.sq_z : w < 0 ? a.sk_z : a.sv_z, y = k < 0 ? a.sq_y : w < 0 ? a.sk_y : a.sv_y;
    const half_t* const from = base + (int64_t)(k < 0 ? h : w < 0 ? k : w) * z + row * y;
    if constexpr (VEC) {
      v = *(const half8_t*)(from + t.x);
      if (t.two) v2 = *(const half8_t*)(from + t.x2);
    } else {
      const int64_t x = k < 0 ? a.sq_x : w < 0 ? a.sk_x : a.sv_x;
      v = from[t.x * x];
      if (t.two) v2 = from[t.x2 * x];
    }
  };
  auto write = [&](const Item& t, int64_t row0, int r, int h) __attribute__((always_inline)) {
    const int k = CACHE ? h - q_heads : -1, w = CACHE ? k - kv_heads : -1;
    const RowPlace p = place[r];
    const int64_t at = k < 0 ? (row0 + r) * a.so_y + h * (int64_t)a.so_z
                             : w < 0 ? p.k + k * a.cache.stride_kz : p.v + w * a.cache.stride_vz;
    if (p.row < 0 || (k >= 0 && (w < 0 ? p.k : p.v) < 0)) return;
    half_t* const to = (k < 0 ? a.q_out : (half_t*)(w < 0 ? a.cache.key : a.cache.value)) + at;
    const float2* const cs = turn + r * half;
    const bool turned = t.pair && w < 0;
    if constexpr (VEC) {
      half8_t o = v, o2 = v2;
      if (turned && a.pairs) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 c = cs[t.in * 4 + e];
          const float xa = (float)v[2 * e], xb = (float)v[2 * e + 1];
          o[2 * e] = (half_t)(xa * c.x - xb * c.y);
          o[2 * e + 1] = (half_t)(xa * c.y + xb * c.x);
        }
      } else if (turned) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 c = cs[t.in * 8 + e];
          const float xa = (float)v[e], xb = (float)v2[e];
          o[e] = (half_t)(xa * c.x - xb * c.y);
          o2[e] = (half_t)(xa * c.y + xb * c.x);
        }
      }
      *(half8_t*)(to + t.x) = o;
      if (t.two) *(half8_t*)(to + t.x2) = o2;
    } else {
      const int64_t x = k < 0 ? a.so_x : w < 0 ? a.cache.stride_kx : a.cache.stride_vx;
      half_t o = v, o2 = v2;
      if (turned) {
        const float2 c = cs[t.in];
        const float xa = (float)v, xb = (float)v2;
        o = (half_t)(xa * c.x - xb * c.y);
        o2 = (half_t)(xa * c.y + xb * c.x);
      }
      to[t.x * x] = o;
      if (t.two) to[t.x2 * x] = o2;
    }
  };

  for (int64_t row0 = (int64_t)blockIdx.x * R;;) {
    const int rows = (int)min((int64_t)R, a.rows - row0);
    for (int r = wave; r < rows; r += 4) {
      const int row = (int)row0 + r;
      RowPlace p = {row, 0, -1, -1};
      if constexpr (CACHE) {
        const int s = sequence_of_row(a.batch.row_offsets, a.batch.sequences, row, lane);
        const int begin = clamp_to(a.batch.row_offsets[s], a.rows), end = clamp_to(a.batch.row_offsets[s + 1], a.rows);
        if (row < begin || row >= end) {
          p.row = -1;
        } else {
          const int64_t x = (int64_t)a.batch.lengths[s] - end + row;
          p.position = (int)x;
          if (x >= 0 && x < (int64_t)a.batch.table_width * a.cache.page_size) {
            const int in_table = (int)x / a.cache.page_size, slot = (int)x - in_table * a.cache.page_size;
            const int page = a.batch.table[(int64_t)s * a.batch.table_pitch + in_table];
            if (page >= 0 && page < a.cache.pages) {
              p.k = page * a.cache.stride_kp + slot * a.cache.stride_ky;
              p.v = page * a.cache.stride_vp + slot * a.cache.stride_vy;
            }
          }
        }
      }
      if (a.positions) p.position = a.positions[row];
      if (lane == 0) place[r] = p;
    }
    __syncthreads();
    for (int i = tid; i < rows * half; i += 256) {
      const int r = i / half, f = i - r * half;
      const double t = (double)place[r].position * a.turns[f];
      float sine, cosine;
      sincospif((float)(2.0 * (t - rint(t))), &sine, &cosine);
      turn[i] = make_float2(cosine * a.magnitude, sine * a.magnitude);
    }
    __syncthreads();
    for (int in = item0; in < items; in += 256) {
      const Item t = item_at(in);
      for (int r = 0, h = first;; h += side_by_side) {
        while (h >= heads) h -= heads, r++;
        if (r >= rows) break;
        read(t, row0 + r, h);
        write(t, row0, r, h);
      }
    }
    row0 += (int64_t)gridDim.x * R;
    if (row0 >= a.rows) break;
    __syncthreads();  // (the next rows' places and angles go where these are read)
  }
}

bool vectors_fit(const RotaryArgs& a) {
  uintptr_t ptrs = 0;
  int64_t strides = 0;
  bool unit = true;
  if (a.q) {
    ptrs |= (uintptr_t)a.q | (uintptr_t)a.q_out;
    strides |= (int64_t)a.so_y | a.so_z | a.sq_y | a.sq_z;
    unit = unit && a.so_x == 1 && a.sq_x == 1;
  }
  if (a.k) {
    const adr_paged_cache& c = a.cache;
    ptrs |= (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)c.key | (uintptr_t)c.value;
    strides |= (int64_t)a.sk_y | a.sk_z | a.sv_y | a.sv_z | c.stride_ky | c.stride_kz | c.stride_kp | c.stride_vy |
               c.stride_vz | c.stride_vp;
    unit = unit && a.sk_x == 1 && a.sv_x == 1 && c.stride_kx == 1 && c.stride_vx == 1;
  }
  return unit && ptrs % 16 == 0 && strides % 8 == 0 && a.d % 8 == 0 && a.dims % (a.pairs ? 8 : 16) == 0;
}

}  // namespace

hipError_t launch_rotary(hipStream_t stream, const RotaryArgs& a) {
  const bool vec = vectors_fit(a);
  const int turned = !vec ? a.dims / 2 : a.pairs ? a.dims / 8 : a.dims / 16;
  const int passing = vec ? (a.d - a.dims) / 8 : a.d - a.dims;
  RotaryJob s = {};
  (RotaryArgs&)s = a;
  s.items = turned + passing;
  const int64_t items = s.items * ((int64_t)(a.q ? a.heads : 0) + 2 * (int64_t)(a.k ? a.kv_heads : 0));
  if (items == 0) return hipSuccess;
  if (items * MAX_ROWS > 0x7fffffff) return hipErrorInvalidConfiguration;
  // Rows of a workgroup: as many as give its 256 threads four items each, within the LDS of their angles, and not so
  // many that there would be fewer than eight workgroups for each of 256 compute units.
  const int half = a.dims / 2;
  int R = (int)std::min<int64_t>(std::max<int64_t>(1024 / items, 1), MAX_ROWS);
  while (R > 1 && (R * half > 2048 || (R * items > 256 && a.rows / R < 2048))) R >>= 1;
  s.rows_per_wg = R;
  const int64_t grid = std::min<int64_t>(((int64_t)a.rows + R - 1) / R, 1 << 22);  // (a launch has fewer than 2^32 threads)
  const size_t lds = MAX_ROWS * sizeof(RowPlace) + (size_t)R * half * sizeof(float2);
  const dim3 blocks((unsigned)grid), threads(256);
  if (vec && a.k) hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<true, true>), blocks, threads, lds, stream, s);
  else if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<true, false>), blocks, threads, lds, stream, s);
  else if (a.k) hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<false, true>), blocks, threads, lds, stream, s);
  else hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_kernel<false, false>), blocks, threads, lds, stream, s);
  return hipGetLastError();
}

}  // namespace adr
