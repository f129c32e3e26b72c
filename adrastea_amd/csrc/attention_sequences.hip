// Attention of packed rows of several sequences, over the pages of a cache or over packed keys.
//
//   out[h, row] = sum_x softmax_x( scale <q[h, row], k[x]> / temp ) v[x],   x <= j + n - r under the mask
//
// for row j of a sequence of r rows and n keys.  Query heads come in groups that share a key and value head.
#include <math.h>

#include <algorithm>

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
    const int64_t room = (int64_t)a.table_width * a.page_size;
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

}  // namespace

SequencesPlan sequences_plan(const SequencesArgs& a, int cus, int64_t avail) {
  (void)a, (void)cus, (void)avail;
  return {0};
}

hipError_t launch_attention_sequences(hipStream_t stream, const SequencesArgs& a, const SequencesPlan& p, void* workspace) {
  (void)p, (void)workspace;
  const int64_t waves = (int64_t)a.rows * a.heads;
  const int64_t grid = std::min<int64_t>((waves + 3) / 4, 1 << 22);
  hipLaunchKernelGGL(attention_any_layout_kernel, dim3((unsigned)grid), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace adr
