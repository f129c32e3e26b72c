// A step's queries, keys and values on their way from the projection: heads normed and turned, keys and values to their
// pages in 16 or in 8 bits; and what is in 8 bits read back.
//
//   y = x / sqrt(mean(x^2) + eps) * weight                                 of each head, queries and keys
//   (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t),          t = 2 pi * position[axis of the pair] * turns[pair]
//   scale = the largest |y| / 127.5, rounded up to fp16;  code = 128 + floor(y / scale), which stands for (code - 127.5) scale
//
// A code is a step of y, and 32 bits would put a y next to a step's border on the wrong side of it now and then: one in
// 10^5 of them.  So what becomes codes is computed in 64 bits (keys; values are fp16, of which 32 bits divide exactly): the codes
// are those of the definition.  Scales are rounded up so that the largest |y| is no more than half a step from its value,
// however small it is; a scale is 513.5 at most, with which all values of codes are finite in fp16.
#include <algorithm>
#include <type_traits>

#include "append.hpp"

namespace adr {
namespace {

enum Cache { NO_CACHE, F16, U8 };

struct PlaceJob : PlaceArgs {
  int lanes;   // that a head needs, of W
  uint32_t first;  // task of the launch
  int splits;  // wavefronts that share a row's heads
};

// ---- sums over the lanes of a head --------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_move(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t other_row(uint32_t v) {  // lane ^ 16
  return (uint32_t)__builtin_amdgcn_ds_swizzle((int)v, 0x401f);
}
template <int STEP, typename T>
__device__ __forceinline__ T partner(T v) {
  static_assert(sizeof(T) % 4 == 0, "");
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 4); i++)  // (of what is equal in both lanes, pairs of lanes ... a mirror is an exchange)
    w[i] = STEP == 1 ? dpp_move<0xb1>(w[i]) : STEP == 2 ? dpp_move<0x4e>(w[i]) : STEP == 4 ? dpp_move<0x141>(w[i])
           : STEP == 8 ? dpp_move<0x140>(w[i]) : other_row(w[i]);
  __builtin_memcpy(&v, w, sizeof(T));
  return v;
}
template <int W, typename T>
__device__ __forceinline__ T sum_of(T v) {
  if constexpr (W > 1) v += partner<1>(v);
  if constexpr (W > 2) v += partner<2>(v);
  if constexpr (W > 4) v += partner<4>(v);
  if constexpr (W > 8) v += partner<8>(v);
  if constexpr (W > 16) v += partner<16>(v);
  return v;
}
__device__ __forceinline__ float absolute(float a) { return fabsf(a); }
__device__ __forceinline__ double absolute(double a) { return fabs(a); }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
template <int W, typename T>
__device__ __forceinline__ T max_of(T v) {
  if constexpr (W > 1) v = larger(v, partner<1>(v));
  if constexpr (W > 2) v = larger(v, partner<2>(v));
  if constexpr (W > 4) v = larger(v, partner<4>(v));
  if constexpr (W > 8) v = larger(v, partner<8>(v));
  if constexpr (W > 16) v = larger(v, partner<16>(v));
  return v;
}

// ---- angles, steps ------------------------------------------------------------------------------------------

// The cosine and sine of `turns` turns a position, times the magnitude.  The product is in 64 bits, its whole turns are taken off
// there, and what is left goes through the 32-bit functions where the result becomes fp16.
template <typename T>
struct Turn {
  T cosine, sine;
};
template <typename T>
__device__ __forceinline__ Turn<T> turn_of(int position, double turns, float magnitude) {
  const double t = (double)position * turns, part = 2.0 * (t - rint(t));
  Turn<T> r;
  if constexpr (sizeof(T) == 8) sincospi(part, &r.sine, &r.cosine);
  else sincospif((float)part, &r.sine, &r.cosine);
  r.cosine *= magnitude, r.sine *= magnitude;
  return r;
}
__device__ __forceinline__ int position_of(const PlaceArgs& a, int row, int pair, int in_cache) {
  if (!a.positions) return in_cache;
  const int axis = a.axis ? a.axis[pair] : 0;
  return a.positions[(int64_t)((unsigned)axis < (unsigned)a.axes ? axis : 0) * a.positions_pitch + row];
}

__device__ __forceinline__ float root(float x) { return sqrtf(x); }
__device__ __forceinline__ double root(double x) { return sqrt(x); }

constexpr float MOST_SCALE = 513.5f;
// The smallest fp16 number that is `top` / 127.5 at least (a comparison of exact products); NaN for what is not finite.
template <typename T>
__device__ __forceinline__ half_t scale_of(T top) {
  if (!(top < (T)INFINITY)) return (half_t)NAN;
  half_t h = (half_t)fminf((float)top * (1.0f / 127.5f), MOST_SCALE);
  uint16_t bits = half_to_bits(h);
  if (bits > 0 && (T)(float)bits_to_half(bits - 1) * (T)127.5 >= top) bits--;
  else if ((T)(float)h * (T)127.5 < top && (float)h < MOST_SCALE) bits++;
  return bits_to_half(bits);
}
__device__ __forceinline__ float step_of(float v) { return floorf(v); }
__device__ __forceinline__ double step_of(double v) { return floor(v); }
__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }
// 128 + floor(y / s), by a product with 1 / s (0 where s is 0 or NaN): that is off by so little that a quotient which is an integer is
// lifted over its border by `lift`, and no other one is.  Quotients of fp16 numbers, of 128 at most, are integers or 2^-12 from the
// next one, and the product in 32 bits is off by 2^-15; in 64 bits those that lie within 2^-40 below an integer are lost.  The
// numbers below 0 that come too near are told by their sign.
template <typename T>
__device__ __forceinline__ uint32_t code_of(T y, T inv) {
  constexpr T lift = sizeof(T) == 8 ? (T)0x1p-40 : (T)0x1p-13;
  const int k = (int)step_of(fused(y, inv, lift));
  return (uint32_t)(min(max(k, -128), y < 0 && inv > 0 ? -1 : 127) + 128);
}
template <typename T>
__device__ __forceinline__ T inverse_of(half_t s) {
  return (float)s > 0.0f ? (T)1 / (T)(float)s : (T)0;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- where a row's key goes -----------------------------------------------------------------------------------

struct Slot {
  int row;        // -1: of no sequence
  int position;   // in the cache
  int page, slot; // page -1: in no page of the cache
};

// Of a row of sequence s, whose rows and keys the batch says to be these.
__device__ __forceinline__ Slot slot_in(const adr_paged_batch& b, int rows, int pages, int page_size, int row, int s, int begin, int end, int length) {
  begin = clamp_to(begin, rows), end = clamp_to(end, rows);
  Slot p = {row, 0, -1, 0};
  if (row < begin || row >= end) {
    p.row = -1;
    return p;
  }
  const int64_t x = (int64_t)length - end + row;
  p.position = (int)x;
  if (x >= 0 && x < (int64_t)b.table_width * page_size) {
    const int at = (int)x / page_size, page = b.table[(int64_t)s * b.table_pitch + at];
    p.slot = (int)x - at * page_size;
    p.page = page >= 0 && page < pages ? page : -1;
  }
  return p;
}

// The sequences of rows first ... last, of which each lane has one, at most a lane's worth of them: one search for the first, and the
// 64 offsets from there on decide for the others.
__device__ __forceinline__ Slot slot_of(const adr_paged_batch& b, int rows, int pages, int page_size, int first, int last, int row, int lane) {
  const int s0 = sequence_of_row(b.row_offsets, b.sequences, first, lane);
  const int ahead = s0 + lane < b.sequences ? b.row_offsets[s0 + lane] : 0x7fffffff;
  int s = s0;
  for (int r = first; r <= last; r++) {
    const int n = __popcll(__ballot(ahead <= r));
    const int at = n < 64 ? s0 + max(n, 1) - 1 : sequence_of_row(b.row_offsets, b.sequences, r, lane);
    if (row == r) s = at;
  }
  return slot_in(b, rows, pages, page_size, row, s, b.row_offsets[s], b.row_offsets[s + 1], b.lengths[s]);
}

// The same of one row, by a wavefront.  Up to 63 sequences are known by one way to memory.
__device__ __forceinline__ Slot slot_of_row(const adr_paged_batch& b, int rows, int pages, int page_size, int row, int lane) {
  int s, begin, end, length;
  if (b.sequences < 64) {
    const int offset = lane <= b.sequences ? b.row_offsets[lane] : 0x7fffffff, of_lane = lane < b.sequences ? b.lengths[lane] : 0;
    s = max(__popcll(__ballot(lane < b.sequences && offset <= row)), 1) - 1;
    begin = __builtin_amdgcn_readlane(offset, s), end = __builtin_amdgcn_readlane(offset, s + 1);
    length = __builtin_amdgcn_readlane(of_lane, s);
  } else {
    s = uniform(sequence_of_row(b.row_offsets, b.sequences, row, lane));
    begin = b.row_offsets[s], end = b.row_offsets[s + 1], length = b.lengths[s];
  }
  return slot_in(b, rows, pages, page_size, row, s, begin, end, length);
}

// ---- 16 bytes at a time -------------------------------------------------------------------------------------

// A wavefront has a row, or shares it with others where rows are few.  W lanes have a head, and the 64 / W heads that a wavefront
// works on lie side by side; a lane has the 16 values that are turned together and so need no exchange: of halves chunk l
// of 8 values and its partner, of pairs two chunks side by side; chunks that pass follow, two to a lane.  Each angle is computed by one
// lane of the wavefront, and comes to the others by way of LDS.
//
// Loads and stores of the loops are under no condition, so that the next head's loads are waited for and not the stores in front
// of them: lanes that are left over do what the last one with values does, and store the same.
//
// Memory bounds it, and how many wavefronts ask for it: a wavefront takes 14 us, nearly all of it waiting, so registers are what counts.
// Angles are read from LDS for every head, weights widened for every head, and a wavefront has one task: kept from head to head, or
// constants from task to task, they made 127 to 187 registers, two or three wavefronts to a SIMD; now 74, six wavefronts, and with codes 107,
// four.  us, then and now: 7008 rows of 32 / 8 heads of 128 into a cache in 16 bits (172 MB) 44.6, 38.2, 4.5 TB/s, where a copy of as many
// bytes has 5.2; 7364 rows of 40 / 8 into one in 8 bits (195 MB) 60.2, 47.9, where the vector ALU is busy 59 % of the time as well; 48
// tokens 5.8, 4.3; one token's queries 3.2, 2.5; 4097 patches of 16 heads of 80 7.8, 6.8.
template <int CACHE, int W>
__global__ __launch_bounds__(256) void place_kernel(PlaceJob a) {
  typedef typename std::conditional<CACHE == U8, double, float>::type angle_t;
  constexpr int GROUPS = 64 / W, MOST_PAIRS = 8 * W;
  __shared__ Turn<float> shared_rounded[4][MOST_PAIRS];
  __shared__ Turn<double> shared_turns[4][CACHE == U8 ? MOST_PAIRS : 1];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), l = min(lane & (W - 1), a.lanes - 1);
  // (pair 8 l + e at e W + l: a lane reads the eight of its l, beside the other lanes'.  Keys that become codes need them in 64 bits.)
  Turn<float>* const rounded = shared_rounded[wave];
  Turn<double>* const turns = shared_turns[wave];
  auto keep = [&](int pair, const Turn<angle_t>& t) __attribute__((always_inline)) {
    const int at = (pair & 7) * W + (pair >> 3);
    rounded[at] = {(float)t.cosine, (float)t.sine};
    if constexpr (CACHE == U8) turns[at] = t;
  };
  const bool mine = (lane & (W - 1)) < a.lanes;
  const int end_q = a.q ? a.heads : 0, end_k = end_q + (CACHE == NO_CACHE ? 0 : a.kv_heads), all = 2 * end_k - end_q;
  // The lane's chunks (first values), and which are turned.
  const int joined = a.pairs ? 0 : a.dims >> 4;
  int x0, x1;
  bool turn0, turn1;
  if (a.pairs) {
    x0 = 16 * l, x1 = x0 + 8;
    turn0 = x0 < a.dims, turn1 = x1 < a.dims;
  } else if (l < joined) {
    x0 = 8 * l, x1 = x0 + (a.dims >> 1);
    turn0 = turn1 = true;
  } else {
    x0 = a.dims + 16 * (l - joined), x1 = x0 + 8;
    turn0 = turn1 = false;
  }
  const bool one = x1 >= a.d;  // (the last of an odd number: its chunk twice)
  if (one) x1 = x0, turn1 = false;
  const float per_value = 1.0f / (float)a.d;
  const int half = a.dims >> 1;
  const uint32_t tasks = (uint32_t)a.rows * a.splits;  // (splits are more than one where there are few rows)
  const uint32_t task = a.first + blockIdx.x * 4 + wave;
  if (task < tasks) {
    const int row = uniform((int)((uint32_t)task / (uint32_t)a.splits)), split = uniform((int)((uint32_t)task - (uint32_t)row * a.splits));
    const int step = GROUPS * a.splits, h0 = split * GROUPS + lane / W;
    // The chunks of a head, asked for a head ahead (behind the last one, that again).
    half8_t n0, n1;
    auto read = [&](int h) __attribute__((always_inline)) {
      const half_t* from = h < end_q ? a.q + h * (int64_t)a.sq_z + row * (int64_t)a.sq_y
                           : h < end_k ? a.k + (h - end_q) * (int64_t)a.sk_z + row * (int64_t)a.sk_y
                                       : a.v + (h - end_k) * (int64_t)a.sv_z + row * (int64_t)a.sv_y;
      n0 = *(const half8_t*)(from + x0);
      n1 = *(const half8_t*)(from + x1);
    };
    read(min(h0, all - 1));
    // Asked for ahead of where the row is: the lane's own angle, and the weights of the first heads.
    const int own_pair = min(lane, max(half - 1, 0));
    const double own_turns = half > 0 ? a.turns[own_pair] : 0.0;
    const int own_axis = half > 0 && a.axis ? a.axis[own_pair] : 0;
    half8_t w0 = {}, w1 = {};
    auto weights = [&](const uint16_t* w) __attribute__((always_inline)) {
      if (w) w0 = *(const half8_t*)(w + x0), w1 = *(const half8_t*)(w + x1);
    };
    weights((const uint16_t*)(end_q > 0 ? a.q_weight : a.k_weight));
    const int own_position =
        a.positions && half > 0 ? a.positions[(int64_t)((unsigned)own_axis < (unsigned)a.axes ? own_axis : 0) * a.positions_pitch + row] : 0;
    Slot at = {row, 0, -1, 0};
    if constexpr (CACHE != NO_CACHE) {
      const int pages = CACHE == U8 ? a.codes.pages : a.cache.pages, size = CACHE == U8 ? a.codes.page_size : a.cache.page_size;
      at = slot_of_row(a.batch, a.rows, pages, size, row, lane);
      if (uniform(at.row) < 0) return;
    }
    if (lane < half) keep(lane, turn_of<angle_t>(a.positions ? own_position : at.position, own_turns, a.magnitude));
    for (int i = lane + 64; i < half; i += 64)
      keep(i, turn_of<angle_t>(position_of(a, row, i, at.position), a.turns[i], a.magnitude));
    __builtin_amdgcn_wave_barrier();
    const int end = CACHE != NO_CACHE && uniform(at.page) < 0 ? end_q : all;  // (keys and values without a slot go nowhere)
    if (h0 >= end) return;

    auto store16 = [&](half_t* to, const half8_t& o0, const half8_t& o1) __attribute__((always_inline)) {
      *(half8_t*)(to + x0) = o0;
      *(half8_t*)(to + x1) = o1;
    };
    // The lane, as a number that the compiler does not know from head to head: what is read by it is read again.
    auto fresh = [&]() __attribute__((always_inline)) {
      int i = l;
      asm volatile("" : "+v"(i));
      return i;
    };
    // Norm and turn 16 values in 32 bits; the norm's factor is applied at the end.
    auto place_rounded = [&](half_t* to, const half8_t& c0, const half8_t& c1, bool norm, float eps)
                             __attribute__((always_inline)) {
      float factor = 1.0f, y[16];
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] = (float)c0[e], y[8 + e] = (float)c1[e];
      if (norm) {
        asm volatile("" : "+v"(w0), "+v"(w1));
        float sum = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) sum = fmaf((float)c0[e], (float)c0[e], sum), sum1 = fmaf((float)c1[e], (float)c1[e], sum1);
        sum = !mine ? 0.0f : one ? sum : sum + sum1;
        factor = __builtin_amdgcn_rsqf(fmaf(sum_of<W>(sum), per_value, eps));
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = fmaf((float)c0[e], (float)w0[e], 0.0f), y[8 + e] = fmaf((float)c1[e], (float)w1[e], 0.0f);
      }
      const int i = fresh();
      // (what passes is not mixed with its neighbour, which may be infinite)
      auto turn = [&](float& u, float& v, int e, bool is_turned) __attribute__((always_inline)) {
        if (e == 4) asm volatile("" ::: "memory");  // (four at a time: eight are six registers more)
        const Turn<float> t = rounded[e * W + i];
        const float x = fmaf(-v, t.sine, u * t.cosine), z = fmaf(v, t.cosine, u * t.sine);
        u = is_turned ? x : u, v = is_turned ? z : v;
      };
      if (a.pairs) {
#pragma unroll
        for (int e = 0; e < 8; e++) turn(y[2 * e], y[2 * e + 1], e, e < 4 ? turn0 : turn1);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) turn(y[e], y[8 + e], e, turn0);
      }
      half8_t o0, o1;
#pragma unroll
      for (int e = 0; e < 8; e++) o0[e] = (half_t)fmaf(y[e], factor, 0.0f), o1[e] = (half_t)fmaf(one ? y[e] : y[8 + e], factor, 0.0f);
      store16(to, o0, o1);
    };
    // 16 values as codes, and the head's scale.
    auto place_codes = [&](auto zero, const auto (&y)[16], uint8_t* codes, half_t* scale) __attribute__((always_inline)) {
      typedef decltype(zero) T;
      T top = 0, none = 0;
#pragma unroll
      for (int e = 0; e < 16; e++) {
        top = larger(top, absolute(y[e]));
        none = fused(y[e], (T)0, none);  // (NaN behind what is not finite)
      }
      top = max_of<W>(top), none = sum_of<W>(none);
      const half_t s = scale_of(none == 0 ? top : (T)INFINITY);
      const T inv = inverse_of<T>(s);
      uint32_t c[4] = {};
#pragma unroll
      for (int e = 0; e < 16; e++) c[e / 4] |= code_of(y[e], inv) << 8 * (e % 4);
      *(u32x2_t*)(codes + x0) = u32x2_t{c[0], c[1]};
      *(u32x2_t*)(codes + x1) = u32x2_t{c[2], c[3]};
      *scale = s;
    };

    int h = h0;
    if (h < min(end, CACHE == F16 ? end_k : end_q)) {
      if (h < end_q) {
        half_t* to = a.q_out + h * (int64_t)a.so_z + row * (int64_t)a.so_y;
        for (; h < end_q; h += step, to += (int64_t)step * a.so_z) {
          const half8_t c0 = n0, c1 = n1;
          read(min(h + step, all - 1));
          place_rounded(to, c0, c1, a.q_weight != nullptr, a.q_eps);
        }
      }
      if (CACHE == F16 && h < min(end, end_k)) {
        weights((const uint16_t*)a.k_weight);
        const adr_paged_cache& c = a.cache;
        half_t* const to = (half_t*)c.key + at.page * c.stride_kp + at.slot * c.stride_ky;
        for (; h < end_k; h += step) {
          const half8_t c0 = n0, c1 = n1;
          read(min(h + step, all - 1));
          place_rounded(to + (h - end_q) * c.stride_kz, c0, c1, a.k_weight != nullptr, a.k_eps);
        }
      }
    }
    if constexpr (CACHE == U8) {
      const adr_paged_cache_u8& c = a.codes;
      if (h < min(end, end_k)) {
        weights((const uint16_t*)a.k_weight);
        uint8_t* const to = c.key + at.page * c.stride_kp + at.slot * c.stride_ky;
        half_t* const scale = (half_t*)c.key_scale + at.page * c.stride_ksp + at.slot * c.stride_ksy;
        for (; h < end_k; h += step) {
          const half8_t c0 = n0, c1 = n1;
          read(min(h + step, all - 1));
          double y[16];
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = (double)(float)c0[e], y[8 + e] = (double)(float)c1[e];
          if (a.k_weight) {
            asm volatile("" : "+v"(w0), "+v"(w1));
            double sum = 0.0, sum1 = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) sum = fma(y[e], y[e], sum), sum1 = fma(y[8 + e], y[8 + e], sum1);
            sum = !mine ? 0.0 : one ? sum : sum + sum1;
            const double factor = 1.0 / sqrt(sum_of<W>(sum) / (double)a.d + (double)a.k_eps);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = y[e] * factor * (double)(float)w0[e], y[8 + e] = y[8 + e] * factor * (double)(float)w1[e];
          }
          const int i = fresh();
          if (a.pairs) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const Turn<double> t = turns[e * W + i];
              const double u = y[2 * e], v = y[2 * e + 1], x = u * t.cosine - v * t.sine, z = u * t.sine + v * t.cosine;
              y[2 * e] = (e < 4 ? turn0 : turn1) ? x : e >= 4 && one ? y[2 * e - 8] : u;
              y[2 * e + 1] = (e < 4 ? turn0 : turn1) ? z : e >= 4 && one ? y[2 * e - 7] : v;
            }
          } else if (turn0) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
              const Turn<double> t = turns[e * W + i];
              const double u = y[e], v = y[8 + e];
              y[e] = u * t.cosine - v * t.sine;
              y[8 + e] = u * t.sine + v * t.cosine;
            }
          }
          place_codes(0.0, y, to + (h - end_q) * c.stride_kz, scale + (h - end_q) * c.stride_ksz);
        }
      }
      uint8_t* const to = c.value + at.page * c.stride_vp + at.slot * c.stride_vy;
      half_t* const scale = (half_t*)c.value_scale + at.page * c.stride_vsp + at.slot * c.stride_vsy;
      for (; h < end; h += step) {
        const half8_t c0 = n0, c1 = n1;
        read(min(h + step, all - 1));
        float y[16];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = (float)c0[e], y[8 + e] = (float)c1[e];
        place_codes(0.0f, y, to + (h - end_k) * c.stride_vz, scale + (h - end_k) * c.stride_vsz);
      }
    }
    if constexpr (CACHE == F16) {
      const adr_paged_cache& c = a.cache;
      half_t* const to = (half_t*)c.value + at.page * c.stride_vp + at.slot * c.stride_vy;
      for (; h < end; h += step) {
        const half8_t c0 = n0, c1 = n1;
        read(min(h + step, all - 1));
        store16(to + (h - end_k) * c.stride_vz, c0, c1);
      }
    }
  }
}

// ---- any layout -----------------------------------------------------------------------------------------------

// A wavefront to a row's head, a lane to every 64th pair or value that passes; values are read again where they are needed again.
template <int CACHE>
__global__ __launch_bounds__(256) void place_any_layout_kernel(PlaceJob a) {
  const int lane = threadIdx.x & 63;
  const int q_heads = a.q ? a.heads : 0, kv_heads = CACHE == NO_CACHE ? 0 : a.kv_heads, all = q_heads + 2 * kv_heads;
  const int half = a.dims >> 1, items = half + a.d - a.dims;
  for (int64_t task = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); task < (int64_t)a.rows * all; task += (int64_t)gridDim.x * 4) {
    const int row = (int)(task / all), h = (int)(task - (int64_t)row * all), k = h - q_heads, v = k - kv_heads;
    Slot at = {row, 0, -1, 0};
    if constexpr (CACHE != NO_CACHE) {
      const int pages = CACHE == U8 ? a.codes.pages : a.cache.pages, size = CACHE == U8 ? a.codes.page_size : a.cache.page_size;
      at = slot_of_row(a.batch, a.rows, pages, size, row, lane);
      if (at.row < 0 || (k >= 0 && at.page < 0)) continue;
    }
    const half_t* const from = k < 0   ? a.q + h * (int64_t)a.sq_z + row * (int64_t)a.sq_y
                               : v < 0 ? a.k + k * (int64_t)a.sk_z + row * (int64_t)a.sk_y
                                       : a.v + v * (int64_t)a.sv_z + row * (int64_t)a.sv_y;
    const int64_t step = k < 0 ? a.sq_x : v < 0 ? a.sk_x : a.sv_x;
    const half_t* const weight = k < 0 ? a.q_weight : v < 0 ? a.k_weight : nullptr;
    const float eps = k < 0 ? a.q_eps : a.k_eps;
    auto go = [&](auto zero) __attribute__((always_inline)) {
      typedef decltype(zero) T;
      T factor = 1;
      if (weight) {
        T sum = 0;
        for (int i = lane; i < a.d; i += 64) sum = fused((T)(float)from[i * step], (T)(float)from[i * step], sum);
        for (int i = 32; i > 0; i >>= 1) sum += __shfl_xor(sum, i);
        factor = (T)1 / root(sum / (T)a.d + (T)eps);
      }
      auto value = [&](int x) __attribute__((always_inline)) {
        const T y = (T)(float)from[x * step];
        return weight ? y * factor * (T)(float)weight[x] : y;
      };
      // Item i: one pair, or one value that passes (of values all do).
      auto each = [&](auto done) __attribute__((always_inline)) {
        for (int i = lane; i < items; i += 64) {
          const int x0 = i >= half ? a.dims + i - half : a.pairs ? 2 * i : i, x1 = i >= half ? -1 : a.pairs ? x0 + 1 : x0 + half;
          T y0 = value(x0), y1 = x1 < 0 ? (T)0 : value(x1);
          if (x1 >= 0 && v < 0) {
            const Turn<T> t = turn_of<T>(position_of(a, row, i, at.position), a.turns[i], a.magnitude);
            const T u = y0;
            y0 = u * t.cosine - y1 * t.sine;
            y1 = u * t.sine + y1 * t.cosine;
          }
          done(x0, y0, x1, y1);
        }
      };
      if (CACHE == U8 && k >= 0) {
        const adr_paged_cache_u8& c = a.codes;
        uint8_t* const to = v < 0 ? c.key + at.page * c.stride_kp + at.slot * c.stride_ky + k * c.stride_kz
                                  : c.value + at.page * c.stride_vp + at.slot * c.stride_vy + v * c.stride_vz;
        half_t* const scale = v < 0 ? (half_t*)c.key_scale + at.page * c.stride_ksp + at.slot * c.stride_ksy + k * c.stride_ksz
                                    : (half_t*)c.value_scale + at.page * c.stride_vsp + at.slot * c.stride_vsy + v * c.stride_vsz;
        const int64_t x_step = v < 0 ? c.stride_kx : c.stride_vx;
        T top = 0, none = 0;
        each([&](int, T y0, int, T y1) __attribute__((always_inline)) {
          top = larger(larger(top, absolute(y0)), absolute(y1));
          none = fused(y0, (T)0, fused(y1, (T)0, none));
        });
        for (int i = 32; i > 0; i >>= 1) top = larger(top, __shfl_xor(top, i)), none += __shfl_xor(none, i);
        const half_t s = scale_of(none == 0 ? top : (T)INFINITY);
        const T inv = inverse_of<T>(s);
        each([&](int i0, T y0, int i1, T y1) __attribute__((always_inline)) {
          to[i0 * x_step] = (uint8_t)code_of(y0, inv);
          if (i1 >= 0) to[i1 * x_step] = (uint8_t)code_of(y1, inv);
        });
        if (lane == 0) *scale = s;
      } else {
        const adr_paged_cache& c = a.cache;
        half_t* const to = k < 0   ? a.q_out + h * (int64_t)a.so_z + row * (int64_t)a.so_y
                           : v < 0 ? (half_t*)c.key + at.page * c.stride_kp + at.slot * c.stride_ky + k * c.stride_kz
                                   : (half_t*)c.value + at.page * c.stride_vp + at.slot * c.stride_vy + v * c.stride_vz;
        const int64_t x_step = k < 0 ? a.so_x : v < 0 ? c.stride_kx : c.stride_vx;
        each([&](int i0, T y0, int i1, T y1) __attribute__((always_inline)) {
          to[i0 * x_step] = (half_t)(float)y0;
          if (i1 >= 0) to[i1 * x_step] = (half_t)(float)y1;
        });
      }
    };
    if (CACHE == U8 && k >= 0 && v < 0) go(0.0);
    else go(0.0f);
  }
}

// ---- reading back -----------------------------------------------------------------------------------------------

struct ReadJob : ReadArgs {
  int items;  // of a row and head, of keys or of values
};

// A thread to an item: 16 codes (VEC), or one.  7364 rows of 8 heads of 128, 46 MB: 14.2 us, 3.2 TB/s, of which start and end are some 4; 64
// tokens 4.3.  Before its codes a wavefront goes to memory four times, one after the other (the search, offsets, length, table), for 1 KB of
// them; the vector ALU is busy 68 % of the time.
template <bool VEC>
__global__ __launch_bounds__(256) void read_u8_kernel(ReadJob a) {
  const adr_paged_cache_u8& c = a.cache;
  const int lane = threadIdx.x & 63, of_row = 2 * c.kv_heads * a.items;
  const int64_t all = (int64_t)a.rows * of_row;
  for (int64_t base = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 64; base < all; base += (int64_t)gridDim.x * 256) {
    const int first = (int)(base / of_row), last = (int)((min(base + 64, all) - 1) / of_row);
    const bool some = base + lane < all;
    const int row = some ? (int)((base + lane) / of_row) : last;
    int in = (int)(base + lane - (int64_t)row * of_row);
    const Slot at = slot_of(a.batch, a.rows, c.pages, c.page_size, first, last, row, lane);
    if (!some || at.row < 0) continue;
    const bool is_v = in >= c.kv_heads * a.items;
    if (is_v) in -= c.kv_heads * a.items;
    const int h = in / a.items, x = (in - h * a.items) * (VEC ? 16 : 1);
    const uint8_t* const codes = is_v ? c.value + at.page * c.stride_vp + at.slot * c.stride_vy + h * c.stride_vz
                                      : c.key + at.page * c.stride_kp + at.slot * c.stride_ky + h * c.stride_kz;
    const half_t* const scale = is_v ? (const half_t*)c.value_scale + at.page * c.stride_vsp + at.slot * c.stride_vsy + h * c.stride_vsz
                                     : (const half_t*)c.key_scale + at.page * c.stride_ksp + at.slot * c.stride_ksy + h * c.stride_ksz;
    half_t* const to = is_v ? a.v + h * (int64_t)a.sv_z + row * (int64_t)a.sv_y : a.k + h * (int64_t)a.sk_z + row * (int64_t)a.sk_y;
    // (a slot on no page is read as NaN; (code - 127.5) scale has 19 bits: one rounding, to fp16)
    if constexpr (VEC) {
      u32x4_t v = {};
      half_t s = (half_t)NAN;
      if (at.page >= 0) v = *(const u32x4_t*)(codes + x), s = *scale;
      const half2_t s2 = {s, s};
      *(half8_t*)(to + x) = dequant8(v[0], v[1], s2);
      *(half8_t*)(to + x + 8) = dequant8(v[2], v[3], s2);
    } else {
      const float s = at.page >= 0 ? (float)*scale : NAN;
      const float v = at.page >= 0 ? (float)codes[x * (is_v ? c.stride_vx : c.stride_kx)] : 0.0f;
      to[x * (int64_t)(is_v ? a.sv_x : a.sk_x)] = (half_t)((v - 127.5f) * s);
    }
  }
}

// Whole chunks of 8 values (codes: 8 bytes) at addresses of their size.
bool vectors_fit(const PlaceArgs& a, Cache cache) {
  uintptr_t ptrs = 0, code_ptrs = 0;
  int64_t strides = 0;
  bool unit = true;
  if (a.q) {
    ptrs |= (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.q_weight;
    strides |= (int64_t)a.so_y | a.so_z | a.sq_y | a.sq_z;
    unit = unit && a.so_x == 1 && a.sq_x == 1;
  }
  if (cache != NO_CACHE) {
    ptrs |= (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_weight;
    strides |= (int64_t)a.sk_y | a.sk_z | a.sv_y | a.sv_z;
    unit = unit && a.sk_x == 1 && a.sv_x == 1;
  }
  if (cache == F16) {
    const adr_paged_cache& c = a.cache;
    ptrs |= (uintptr_t)c.key | (uintptr_t)c.value;
    strides |= c.stride_ky | c.stride_kz | c.stride_kp | c.stride_vy | c.stride_vz | c.stride_vp;
    unit = unit && c.stride_kx == 1 && c.stride_vx == 1;
  } else if (cache == U8) {
    const adr_paged_cache_u8& c = a.codes;
    code_ptrs |= (uintptr_t)c.key | (uintptr_t)c.value;
    strides |= c.stride_ky | c.stride_kz | c.stride_kp | c.stride_vy | c.stride_vz | c.stride_vp;
    unit = unit && c.stride_kx == 1 && c.stride_vx == 1;
  }
  return unit && ptrs % 16 == 0 && code_ptrs % 8 == 0 && strides % 8 == 0 && a.d % 8 == 0 && a.d <= 512 &&
         a.dims % (a.pairs ? 8 : 16) == 0;
}

template <int CACHE>
hipError_t launch_place_into(hipStream_t stream, const PlaceArgs& a) {
  PlaceJob job = {};
  (PlaceArgs&)job = a;
  const int64_t heads = (int64_t)(a.q ? a.heads : 0) + (CACHE == NO_CACHE ? 0 : 2 * (int64_t)a.kv_heads);
  if (heads > 0x7fffffff) return hipErrorInvalidConfiguration;
  constexpr int64_t MOST = 1 << 22;  // workgroups (a launch has fewer than 2^32 threads)
  if (!vectors_fit(a, (Cache)CACHE)) {
    const unsigned grid = (unsigned)std::min<int64_t>(((int64_t)a.rows * heads + 3) / 4, MOST);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(place_any_layout_kernel<CACHE>), dim3(grid), dim3(256), 0, stream, job);
    return hipGetLastError();
  }
  const int lanes = a.pairs ? (a.d + 15) / 16 : a.dims / 16 + (a.d - a.dims + 15) / 16;
  job.lanes = lanes;
  const int W = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : 32;
  // Wavefronts that share a row: one for each of its steps where there are few rows, fewer where the rows alone make 16
  // wavefronts for each of 256 compute units.
  const int64_t steps = (heads + 64 / W - 1) / (64 / W);
  job.splits = (int)std::min<int64_t>(std::max<int64_t>((256 * 16 + a.rows - 1) / a.rows, 1), steps);
  const int64_t tasks = (int64_t)a.rows * job.splits;
  for (int64_t first = 0; first < tasks; first += 4 * MOST) {
    job.first = (uint32_t)first;
    const unsigned grid = (unsigned)std::min<int64_t>((tasks - first + 3) / 4, MOST);
    if (W == 4) hipLaunchKernelGGL(HIP_KERNEL_NAME(place_kernel<CACHE, 4>), dim3(grid), dim3(256), 0, stream, job);
    else if (W == 8) hipLaunchKernelGGL(HIP_KERNEL_NAME(place_kernel<CACHE, 8>), dim3(grid), dim3(256), 0, stream, job);
    else if (W == 16) hipLaunchKernelGGL(HIP_KERNEL_NAME(place_kernel<CACHE, 16>), dim3(grid), dim3(256), 0, stream, job);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(place_kernel<CACHE, 32>), dim3(grid), dim3(256), 0, stream, job);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_place(hipStream_t stream, const PlaceArgs& a) {
  if (!a.k) return launch_place_into<NO_CACHE>(stream, a);
  return a.in_codes ? launch_place_into<U8>(stream, a) : launch_place_into<F16>(stream, a);
}

hipError_t launch_read_u8(hipStream_t stream, const ReadArgs& a) {
  const adr_paged_cache_u8& c = a.cache;
  const uintptr_t ptrs = (uintptr_t)c.key | (uintptr_t)c.value | (uintptr_t)a.k | (uintptr_t)a.v;
  const int64_t strides = c.stride_ky | c.stride_kz | c.stride_kp | c.stride_vy | c.stride_vz | c.stride_vp;
  const int64_t out = (int64_t)a.sk_y | a.sk_z | a.sv_y | a.sv_z;
  const bool vec = ptrs % 16 == 0 && strides % 16 == 0 && out % 8 == 0 && c.d % 16 == 0 && a.sk_x == 1 && a.sv_x == 1 &&
                   c.stride_kx == 1 && c.stride_vx == 1;
  ReadJob job = {};
  (ReadArgs&)job = a;
  job.items = vec ? c.d / 16 : c.d;
  if (2 * (int64_t)c.kv_heads * job.items > 0x7fffffff) return hipErrorInvalidConfiguration;
  const unsigned grid = (unsigned)std::min<int64_t>(((int64_t)a.rows * 2 * c.kv_heads * job.items + 255) / 256, 1 << 22);
  if (vec) hipLaunchKernelGGL(HIP_KERNEL_NAME(read_u8_kernel<true>), dim3(grid), dim3(256), 0, stream, job);
  else hipLaunchKernelGGL(HIP_KERNEL_NAME(read_u8_kernel<false>), dim3(grid), dim3(256), 0, stream, job);
  return hipGetLastError();
}

}  // namespace adr
