// Rotary positions, and a step's new keys and values into the pages of the cache.
//
//   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),   t = 2 pi * position * turns[i]
//
// The angle is made where it is used: a table of cosines would be read from memory for every row and has an
// end.  position * turns[i] is a 64-bit product (positions of seven digits leave 2^-33 of a turn), its whole
// turns are taken off in 64 bits, and what is left, at most half a turn, goes through the 32-bit sincospi.
// Each is computed once per row and pair, by a thread of its own, and shared by all heads through LDS.
#include <algorithm>

#include "sequences.hpp"

namespace adr {
namespace {

constexpr int MAX_ROWS = 16;  // of a workgroup

struct RowPlace {   // of one row of the workgroup
  int row;          // -1: none
  int position;
  int64_t k, v;     // element offset of its slot in the cache (head 0); -1: not written
};

// The grid's geometry, chosen by the host.
struct RotaryShape {
  int rows_per_wg;
  int q_items, k_items, v_items;  // work items of one head: 8 or 16 values, or one or two
  int row_items;                  // of a row
};

// VEC: 16 bytes at a time -- one item is a pair of chunks of 8 values (halves), a chunk of 4 pairs (pairs), or
// a chunk that passes.  Otherwise an item is one pair or one value that passes, at any stride.
template <bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, RotaryShape shape) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  RowPlace* const place = (RowPlace*)smem;                                     // [rows_per_wg]
  float2* const turn = (float2*)(smem + MAX_ROWS * sizeof(RowPlace));          // [rows_per_wg][dims / 2]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int R = shape.rows_per_wg, half = a.dims >> 1;

  for (int64_t row0 = (int64_t)blockIdx.x * R; row0 < a.rows; row0 += (int64_t)gridDim.x * R) {
  for (int r = wave; r < R; r += 4) {
    RowPlace p = {-1, 0, -1, -1};
    const int64_t row64 = row0 + r;
    if (row64 < a.rows) {
      const int row = (int)row64;
      p.row = row;
      if (a.k) {
        const int s = sequence_of_row(a.batch.row_offsets, a.batch.sequences, row, lane);
        const int first = clamp_to(a.batch.row_offsets[s], a.rows), end = clamp_to(a.batch.row_offsets[s + 1], a.rows);
        if (row < first || row >= end) {
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
    }
    if (lane == 0) place[r] = p;
  }
  __syncthreads();
  for (int i = tid; i < R * half; i += 256) {
    const int r = i / half, f = i - r * half;
    const double t = (double)place[r].position * a.turns[f];
    float sine, cosine;
    sincospif((float)(2.0 * (t - rint(t))), &sine, &cosine);
    turn[i] = make_float2(cosine * a.magnitude, sine * a.magnitude);
  }
  __syncthreads();

  const int q_all = a.heads * shape.q_items, k_all = a.kv_heads * shape.k_items;
  for (int i = tid; i < R * shape.row_items; i += 256) {
    const int r = i / shape.row_items;
    int item = i - r * shape.row_items;
    const RowPlace p = place[r];
    if (p.row < 0) continue;
    const half_t* src;
    half_t* dst;
    int64_t src_x, dst_x;
    bool rotated = true;
    if (item < q_all) {
      const int h = item / shape.q_items;
      item -= h * shape.q_items;
      src = a.q + (int64_t)h * a.sq_z + (int64_t)p.row * a.sq_y;
      dst = a.q_out + (int64_t)h * a.so_z + (int64_t)p.row * a.so_y;
      src_x = a.sq_x, dst_x = a.so_x;
    } else if (item < q_all + k_all) {
      item -= q_all;
      const int h = item / shape.k_items;
      item -= h * shape.k_items;
      if (p.k < 0) continue;
      src = a.k + (int64_t)h * a.sk_z + (int64_t)p.row * a.sk_y;
      dst = (half_t*)a.cache.key + p.k + h * a.cache.stride_kz;
      src_x = a.sk_x, dst_x = a.cache.stride_kx;
    } else {
      item -= q_all + k_all;
      const int h = item / shape.v_items;
      item -= h * shape.v_items;
      if (p.v < 0) continue;
      src = a.v + (int64_t)h * a.sv_z + (int64_t)p.row * a.sv_y;
      dst = (half_t*)a.cache.value + p.v + h * a.cache.stride_vz;
      src_x = a.sv_x, dst_x = a.cache.stride_vx;
      rotated = false;
    }
    const float2* const cs = turn + r * half;
    if constexpr (VEC) {
      const int turned = !rotated ? 0 : a.pairs ? a.dims >> 3 : a.dims >> 4;  // items of this head that are turned
      if (item >= turned) {
        const int x = (rotated ? a.dims : 0) + (item - turned) * 8;
        *(half8_t*)(dst + x) = *(const half8_t*)(src + x);
      } else if (a.pairs) {
        const half8_t v = *(const half8_t*)(src + item * 8);
        half8_t o;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float2 t = cs[item * 4 + e];
          const float x = (float)v[2 * e], y = (float)v[2 * e + 1];
          o[2 * e] = (half_t)(x * t.x - y * t.y);
          o[2 * e + 1] = (half_t)(x * t.y + y * t.x);
        }
        *(half8_t*)(dst + item * 8) = o;
      } else {
        const half8_t va = *(const half8_t*)(src + item * 8), vb = *(const half8_t*)(src + half + item * 8);
        half8_t oa, ob;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float2 t = cs[item * 8 + e];
          const float x = (float)va[e], y = (float)vb[e];
          oa[e] = (half_t)(x * t.x - y * t.y);
          ob[e] = (half_t)(x * t.y + y * t.x);
        }
        *(half8_t*)(dst + item * 8) = oa;
        *(half8_t*)(dst + half + item * 8) = ob;
      }
    } else {
      if (!rotated || item >= half) {
        const int x = rotated ? item - half + a.dims : item;
        dst[x * dst_x] = src[x * src_x];
      } else {
        const int xa = a.pairs ? 2 * item : item, xb = a.pairs ? xa + 1 : item + half;
        const float2 t = cs[item];
        const float x = (float)src[xa * src_x], y = (float)src[xb * src_x];
        dst[xa * dst_x] = (half_t)(x * t.x - y * t.y);
        dst[xb * dst_x] = (half_t)(x * t.y + y * t.x);
      }
    }
  }
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
  // (in place, what passes is there already)
  const bool in_place = a.q == a.q_out && a.sq_x == a.so_x && a.sq_y == a.so_y && a.sq_z == a.so_z;
  RotaryShape s = {};
  s.q_items = a.q ? turned + (in_place ? 0 : passing) : 0;
  s.k_items = a.k ? turned + passing : 0;
  s.v_items = a.k ? (vec ? a.d / 8 : a.d) : 0;
  const int64_t items = (int64_t)a.heads * s.q_items + (int64_t)a.kv_heads * (s.k_items + s.v_items);
  if (items == 0) return hipSuccess;
  if (items * MAX_ROWS > 0x7fffffff) return hipErrorInvalidConfiguration;
  s.row_items = (int)items;
  // Rows of a workgroup: as many as give its 256 threads an item each, within the LDS of their angles.
  const int half = a.dims / 2;
  int R = (int)std::min<int64_t>(std::max<int64_t>(256 / items, 1), a.k ? 4 : MAX_ROWS);
  while (R > 1 && R * half > 2048) R >>= 1;
  s.rows_per_wg = R;
  const int64_t grid = std::min<int64_t>(((int64_t)a.rows + R - 1) / R, 1 << 22);  // (a launch has fewer than 2^32 threads)
  const size_t lds = MAX_ROWS * sizeof(RowPlace) + (size_t)R * half * sizeof(float2);
  if (vec) hipLaunchKernelGGL(rotary_kernel<true>, dim3((unsigned)grid), dim3(256), lds, stream, a, s);
  else hipLaunchKernelGGL(rotary_kernel<false>, dim3((unsigned)grid), dim3(256), lds, stream, a, s);
  return hipGetLastError();
}

}  // namespace adr
