// The arguments of append.hip: a step's heads normed, turned and put to their places, and codes read back.
#pragma once

#include "sequences.hpp"

namespace adr {

struct PlaceArgs {
  half_t* q_out;
  const half_t* q;  // null: keys and values only
  int so_x, so_y, so_z, sq_x, sq_y, sq_z;
  const half_t* k;  // null: queries only
  const half_t* v;
  int sk_x, sk_y, sk_z, sv_x, sv_y, sv_z;
  const int* positions;  // [axes][rows]; null: positions in the cache
  int positions_pitch;
  const double* turns;
  const int* axis;  // of each pair; null: the first
  int axes, dims, pairs;  // pairs: ADR_ROTARY_PAIRS
  float magnitude;
  const half_t* q_weight;  // null: not normed
  const half_t* k_weight;
  float q_eps, k_eps;
  int heads, kv_heads, rows, d;
  bool in_codes;  // the cache is `codes`
  adr_paged_cache cache;
  adr_paged_cache_u8 codes;
  adr_paged_batch batch;
};
hipError_t launch_place(hipStream_t stream, const PlaceArgs& a);

struct ReadArgs {
  half_t* k;
  half_t* v;
  int sk_x, sk_y, sk_z, sv_x, sv_y, sv_z;
  int rows;
  adr_paged_cache_u8 cache;
  adr_paged_batch batch;
};
hipError_t launch_read_u8(hipStream_t stream, const ReadArgs& a);

}  // namespace adr
