// C++ host side of the matmul interface, mirroring adrastea_models/src/kernels.rs:81-167
// (option types), :206-213 (the two trait methods), :753-890 (lowering to the 22-scalar tuple)
// and :231-359 (MatmulTracer).  GpuKernels launches through the C ABI of
// include/adrastea_kernels.h; shape mismatches throw std::logic_error where the reference
// assert_eq!-panics, launcher errors throw AdrasteaError where it returns anyhow::Error.
#pragma once

#include <mutex>
#include <set>
#include <stdexcept>
#include <string>
#include <tuple>

#include "../../include/adrastea_kernels.h"
#include "tensor.hpp"

namespace adrastea {

using f16 = uint16_t;  // raw fp16 bits

struct AdrasteaError : std::runtime_error {
  int code;
  AdrasteaError(int c, const std::string& what) : std::runtime_error(what + ": " + adr_strerror(c)), code(c) {}
};

enum class MatmulMask : uint32_t { None = 0, Causal = 1 };

struct MatmulLoad {
  uint32_t op = ADR_LOAD_IDENTITY;
  float scale = 1.0f;
  static MatmulLoad Identity() { return {}; }
  static MatmulLoad Scale(float s) { return {ADR_LOAD_SCALE, s}; }
  uint32_t lower() const { return op; }
};

struct MatmulStore {
  uint32_t op = ADR_STORE_IDENTITY;
  float beta = 0.0f, scale = 1.0f;
  const f16* bias = nullptr;  // length-N vector indexed by output column
  static MatmulStore Identity() { return {}; }
  static MatmulStore GeluBias(const f16* b) { return {ADR_STORE_GELU_BIAS, 0, 1, b}; }
  static MatmulStore QuickGeluBias(const f16* b) { return {ADR_STORE_QUICK_GELU_BIAS, 0, 1, b}; }
  static MatmulStore BetaGeluBias(float beta, const f16* b) { return {ADR_STORE_BETA_GELU_BIAS, beta, 1, b}; }
  static MatmulStore BetaBias(float beta, const f16* b) { return {ADR_STORE_BETA_BIAS, beta, 1, b}; }
  static MatmulStore Scale(float s) { return {ADR_STORE_SCALE, 0, s, nullptr}; }
  static MatmulStore Add() { return {ADR_STORE_ADD, 0, 1, nullptr}; }
  uint32_t lower() const { return op; }
};

struct MatmulOptions {
  MatmulLoad load_;
  MatmulStore store_;
  MatmulMask mask_ = MatmulMask::None;
  static MatmulOptions make() { return {}; }
  MatmulOptions load(MatmulLoad l) const { MatmulOptions o = *this; o.load_ = l; return o; }
  MatmulOptions store(MatmulStore s) const { MatmulOptions o = *this; o.store_ = s; return o; }
  MatmulOptions mask(MatmulMask m) const { MatmulOptions o = *this; o.mask_ = m; return o; }
};

struct LoweredMatmul {
  int32_t batches, m, k, n;
  int32_t so[3], sl[3], sr[3];  // (x, y, z) strides of output, left, right
  float beta, scale;
  uint32_t store, load, mask;
};

inline LoweredMatmul lower_matmul(const TensorLayout& out, const TensorLayout& left, const TensorLayout& right,
                                  const MatmulOptions& o) {
  if (left.size(-1) != right.size(-2)) throw std::logic_error("K mismatch");   // kernels.rs:825
  if (out.size(-2) != left.size(-2)) throw std::logic_error("M mismatch");     // kernels.rs:826
  if (out.size(-1) != right.size(-1)) throw std::logic_error("N mismatch");    // kernels.rs:827
  LoweredMatmul r{};
  float scale = o.load_.op == ADR_LOAD_SCALE ? o.load_.scale : 1.0f;
  if (o.store_.op == ADR_STORE_SCALE) scale *= o.store_.scale;  // ONE float for both (:837-843)
  r.scale = scale;
  r.beta = (o.store_.op == ADR_STORE_BETA_GELU_BIAS || o.store_.op == ADR_STORE_BETA_BIAS) ? o.store_.beta : 0.0f;
  r.batches = out.dims.size() > 2 ? (int32_t)out.size(-3) : 1;
  r.m = (int32_t)left.size(-2); r.k = (int32_t)left.size(-1); r.n = (int32_t)right.size(-1);
  auto xyz = [](const TensorLayout& l, int32_t* s) {
    s[0] = (int32_t)l.stride(-1); s[1] = (int32_t)l.stride(-2);
    s[2] = l.dims.size() > 2 ? (int32_t)l.stride(-3) : 0;  // rank-2 operands broadcast (:868-880)
  };
  xyz(out, r.so); xyz(left, r.sl); xyz(right, r.sr);
  r.store = o.store_.lower(); r.load = o.load_.lower(); r.mask = (uint32_t)o.mask_;
  return r;
}

// ---- several sequences at once (not in the reference) ----

// A size or a stride as the C ABI takes it; strides of a dimension of one are never used, and may be anything.
inline int32_t int32_of(size_t v, const char* what, bool used = true) {
  const int64_t x = (int64_t)v;
  if (x >= INT32_MIN && x <= INT32_MAX) return (int32_t)x;
  if (used) throw std::logic_error(std::string(what) + ": " + std::to_string(x) + " does not fit 32 bits");
  return 0;
}

// Keys and values of many sequences in pages: [pages, kv_heads, page_size, d] views of the caller's pools.
struct PagedCache {
  TensorView<f16> key, value;
  adr_paged_cache lower() const {
    const auto &k = key.layout, &v = value.layout;
    if (k.dims.size() != 4 || k.dims != v.dims) throw std::logic_error("PagedCache: [pages, kv_heads, page_size, d] views");
    adr_paged_cache c{};
    c.key = key.ptr, c.value = value.ptr;
    auto size = [&](int i) { return int32_of(k.dims[i], "PagedCache"); };
    c.pages = size(0), c.kv_heads = size(1), c.page_size = size(2), c.d = size(3);
    c.stride_kx = (int64_t)k.strides[3], c.stride_ky = (int64_t)k.strides[2], c.stride_kz = (int64_t)k.strides[1], c.stride_kp = (int64_t)k.strides[0];
    c.stride_vx = (int64_t)v.strides[3], c.stride_vy = (int64_t)v.strides[2], c.stride_vz = (int64_t)v.strides[1], c.stride_vp = (int64_t)v.strides[0];
    return c;
  }
};
// Device memory of the caller: see adr_paged_batch and adr_packed_batch.
using PagedBatch = adr_paged_batch;
using PackedBatch = adr_packed_batch;
using Rotary = adr_rotary;
using RotaryAxes = adr_rotary_axes;
using HeadNorm = adr_head_norm;
using DraftTree = adr_draft_tree;

// Keys and values in 8 bits: [pages, kv_heads, page_size, d] views of codes and [pages, kv_heads, page_size] views of their scales.
struct PagedCacheU8 {
  TensorView<uint8_t> key;
  TensorView<f16> key_scale;
  TensorView<uint8_t> value;
  TensorView<f16> value_scale;
  adr_paged_cache_u8 lower() const {
    const auto &k = key.layout, &v = value.layout, &ks = key_scale.layout, &vs = value_scale.layout;
    if (k.dims.size() != 4 || k.dims != v.dims) throw std::logic_error("PagedCacheU8: [pages, kv_heads, page_size, d] views");
    const std::vector<size_t> scales(k.dims.begin(), k.dims.end() - 1);
    if (ks.dims != scales || vs.dims != scales) throw std::logic_error("PagedCacheU8: [pages, kv_heads, page_size] views of scales");
    adr_paged_cache_u8 c{};
    c.key = key.ptr, c.key_scale = key_scale.ptr, c.value = value.ptr, c.value_scale = value_scale.ptr;
    auto size = [&](int i) { return int32_of(k.dims[i], "PagedCacheU8"); };
    c.pages = size(0), c.kv_heads = size(1), c.page_size = size(2), c.d = size(3);
    c.stride_kx = (int64_t)k.strides[3], c.stride_ky = (int64_t)k.strides[2], c.stride_kz = (int64_t)k.strides[1], c.stride_kp = (int64_t)k.strides[0];
    c.stride_vx = (int64_t)v.strides[3], c.stride_vy = (int64_t)v.strides[2], c.stride_vz = (int64_t)v.strides[1], c.stride_vp = (int64_t)v.strides[0];
    c.stride_ksy = (int64_t)ks.strides[2], c.stride_ksz = (int64_t)ks.strides[1], c.stride_ksp = (int64_t)ks.strides[0];
    c.stride_vsy = (int64_t)vs.strides[2], c.stride_vsz = (int64_t)vs.strides[1], c.stride_vsp = (int64_t)vs.strides[0];
    return c;
  }
};

// What a step appends: its keys and values, its queries with the view that they are turned into (both null: none), the positions on
// each axis (device memory, `pitch` entries from axis to axis, 0: the same for all; null: the places in the cache), the rotation and the norms.
struct Appended {
  TensorView<const f16> key, value;
  RotaryAxes rotary{nullptr, nullptr, 0, ADR_ROTARY_HALVES, 1.0f, 1};
  HeadNorm query_norm{}, key_norm{};
  TensorView<f16>* query_out = nullptr;
  const TensorView<const f16>* query = nullptr;
  const int32_t* positions = nullptr;
  int32_t pitch = 0;
};

struct CommonKernels {
  virtual ~CommonKernels() = default;
  virtual void matmul_f16(TensorView<f16>& output, const TensorView<const f16>& left,
                          const TensorView<const f16>& right, const MatmulOptions& options) = 0;
  virtual void matmul_f16_slow(TensorView<f16>& output, const TensorView<const f16>& left,
                               const TensorView<const f16>& right, const MatmulOptions& options) = 0;
  virtual void softmax_rows_inplace(TensorView<f16>& output, float temperature) = 0;
  // Not in the reference's trait: the three calls of llama.rs:541-554 (QK^T with Scale and the
  // mask, softmax_rows_inplace, P.V) as one launch.  query/output: [heads, m, d] views, key/value:
  // [heads, n, d] views (rank 2 = one head).
  virtual void attention_f16(TensorView<f16>& output, const TensorView<const f16>& query,
                             const TensorView<const f16>& key, const TensorView<const f16>& value,
                             float scale, float temperature, MatmulMask mask) = 0;
  virtual void error_stats_f16(TensorView<float>& output, const TensorView<const f16>& lhs,
                               const TensorView<const f16>& rhs) = 0;
  virtual void error_stats_f32(TensorView<float>& output, const TensorView<const float>& lhs,
                               const TensorView<const float>& rhs) = 0;
  // Several sequences at once (an interface of its own, for implementations that offer it): see adr_rotary_f16,
  // adr_append_f16, adr_attention_paged_f16 and adr_attention_packed_f16.
  // The rows of `input` turned by positions[row] (device memory, [rows]) into `output`, which may be the same view.
  virtual void rotary_f16(TensorView<f16>& /*output*/, const TensorView<const f16>& /*input*/, const int32_t* /*positions*/,
                          const Rotary& /*rotary*/) {
    throw AdrasteaError(ADR_ENOTIMPL, "rotary_f16");
  }
  // The step's keys, turned, and values into their pages, and its queries turned into `query_out` (both null: none).
  virtual void append_f16(const PagedCache& /*cache*/, const PagedBatch& /*batch*/, const TensorView<const f16>& /*key*/,
                          const TensorView<const f16>& /*value*/, const Rotary& /*rotary*/, TensorView<f16>* /*query_out*/ = nullptr,
                          const TensorView<const f16>* /*query*/ = nullptr, const int32_t* /*positions*/ = nullptr) {
    throw AdrasteaError(ADR_ENOTIMPL, "append_f16");
  }
  virtual void attention_paged_f16(TensorView<f16>& /*output*/, const TensorView<const f16>& /*query*/, const PagedCache& /*cache*/,
                                   const PagedBatch& /*batch*/, float /*scale*/, float /*temperature*/ = 1.0f,
                                   MatmulMask /*mask*/ = MatmulMask::Causal) {
    throw AdrasteaError(ADR_ENOTIMPL, "attention_paged_f16");
  }
  virtual void attention_packed_f16(TensorView<f16>& /*output*/, const TensorView<const f16>& /*query*/,
                                    const TensorView<const f16>& /*key*/, const TensorView<const f16>& /*value*/,
                                    const PackedBatch& /*batch*/, float /*scale*/, float /*temperature*/ = 1.0f,
                                    MatmulMask /*mask*/ = MatmulMask::Causal) {
    throw AdrasteaError(ADR_ENOTIMPL, "attention_packed_f16");
  }
  // Heads normed and turned on several axes, a cache in 8 bits, drafted trees: see adr_norm_rotary_f16, adr_append_norm_f16,
  // adr_append_u8, adr_read_u8, adr_attention_paged_u8, adr_attention_tree_f16 and adr_attention_tree_u8.
  // The heads of `input` normed and turned into `output`, which may be the same view; positions [axes][pitch].
  virtual void norm_rotary_f16(TensorView<f16>& /*output*/, const TensorView<const f16>& /*input*/, const int32_t* /*positions*/,
                               int32_t /*pitch*/, const RotaryAxes& /*rotary*/, const HeadNorm& /*norm*/) {
    throw AdrasteaError(ADR_ENOTIMPL, "norm_rotary_f16");
  }
  virtual void append_norm_f16(const PagedCache& /*cache*/, const PagedBatch& /*batch*/, const Appended& /*step*/) {
    throw AdrasteaError(ADR_ENOTIMPL, "append_norm_f16");
  }
  virtual void append_u8(const PagedCacheU8& /*cache*/, const PagedBatch& /*batch*/, const Appended& /*step*/) {
    throw AdrasteaError(ADR_ENOTIMPL, "append_u8");
  }
  // What the codes of the batch's rows stand for.
  virtual void read_u8(TensorView<f16>& /*key_out*/, TensorView<f16>& /*value_out*/, const PagedCacheU8& /*cache*/, const PagedBatch& /*batch*/) {
    throw AdrasteaError(ADR_ENOTIMPL, "read_u8");
  }
  virtual void attention_paged_u8(TensorView<f16>& /*output*/, const TensorView<const f16>& /*query*/, const PagedCacheU8& /*cache*/,
                                  const PagedBatch& /*batch*/, float /*scale*/, float /*temperature*/ = 1.0f,
                                  MatmulMask /*mask*/ = MatmulMask::Causal) {
    throw AdrasteaError(ADR_ENOTIMPL, "attention_paged_u8");
  }
  virtual void attention_tree_f16(TensorView<f16>& /*output*/, const TensorView<const f16>& /*query*/, const PagedCache& /*cache*/,
                                  const PagedBatch& /*batch*/, const DraftTree& /*tree*/, float /*scale*/, float /*temperature*/ = 1.0f) {
    throw AdrasteaError(ADR_ENOTIMPL, "attention_tree_f16");
  }
  virtual void attention_tree_u8(TensorView<f16>& /*output*/, const TensorView<const f16>& /*query*/, const PagedCacheU8& /*cache*/,
                                 const PagedBatch& /*batch*/, const DraftTree& /*tree*/, float /*scale*/, float /*temperature*/ = 1.0f) {
    throw AdrasteaError(ADR_ENOTIMPL, "attention_tree_u8");
  }
};

// TensorGpuDescriptor::from (kernels.rs:38-55): dims and strides reversed, innermost first.
template <typename T>
inline adr_tensor_desc descriptor(const TensorView<T>& v) {
  adr_tensor_desc d{};
  d.ptr = (void*)v.ptr;
  d.dims = (uint32_t)v.layout.dims.size();
  for (size_t i = 0; i < v.layout.dims.size(); i++) {
    d.shape[i] = (uint32_t)v.layout.dims[v.layout.dims.size() - 1 - i];
    d.strides[i] = (uint32_t)v.layout.strides[v.layout.dims.size() - 1 - i];
  }
  return d;
}

class GpuKernels : public CommonKernels {
 public:
  // `workspace`: optional device buffer (16-byte aligned) the caller owns for as long as this
  // object lives; with it, products with few output tiles and a long K are split over K
  // (adr_matmul_f16_ws) and the keys of few query rows shared (adr_attention_f16_ws).  Calls on one object must not overlap in time when it is set.
  explicit GpuKernels(adr_stream_t stream = nullptr, void* workspace = nullptr, int64_t workspace_bytes = 0)
      : stream_(stream), workspace_(workspace), workspace_bytes_(workspace ? workspace_bytes : 0) {}
  void matmul_f16(TensorView<f16>& o, const TensorView<const f16>& l, const TensorView<const f16>& r,
                  const MatmulOptions& opt) override {
    if (workspace_bytes_ <= 0) return run(adr_matmul_f16, "matmul_f16", o, l, r, opt);
    LoweredMatmul w = lower_matmul(o.layout, l.layout, r.layout, opt);
    int rc = adr_matmul_f16_ws(stream_, o.ptr, l.ptr, r.ptr, w.batches, w.m, w.k, w.n, w.so[0], w.so[1], w.so[2],
                               w.sl[0], w.sl[1], w.sl[2], w.sr[0], w.sr[1], w.sr[2], opt.store_.bias, w.beta,
                               w.scale, w.store, w.load, w.mask, workspace_, workspace_bytes_);
    if (rc) throw AdrasteaError(rc, "matmul_f16");
  }
  void matmul_f16_slow(TensorView<f16>& o, const TensorView<const f16>& l, const TensorView<const f16>& r,
                       const MatmulOptions& opt) override { run(adr_matmul_f16_slow, "matmul_f16_slow", o, l, r, opt); }
  // kernels.rs:892-915: rows = size(-2), heads = size(-3) (1 for rank 2), width = size(-1); like
  // the reference's kernel, the view is taken to be contiguous.
  void softmax_rows_inplace(TensorView<f16>& o, float temperature) override {
    if (!(o.layout == TensorLayout::row_major(o.layout.dims))) throw std::logic_error("softmax_rows: contiguous view");
    const int32_t heads = o.layout.dims.size() > 2 ? (int32_t)o.size(-3) : 1;
    int rc = adr_softmax_rows(stream_, o.ptr, o.ptr, heads, (int32_t)o.size(-2), (int32_t)o.size(-1), temperature);
    if (rc) throw AdrasteaError(rc, "softmax_rows_inplace");
  }
  void attention_f16(TensorView<f16>& o, const TensorView<const f16>& q, const TensorView<const f16>& k,
                     const TensorView<const f16>& v, float scale, float temperature, MatmulMask mask) override {
    const size_t rank = q.layout.dims.size();
    if ((rank != 2 && rank != 3) || o.layout.dims.size() != rank || k.layout.dims.size() != rank ||
        v.layout.dims.size() != rank)
      throw std::logic_error("attention_f16: rank 2 or 3 views");
    const int32_t heads = rank == 3 ? (int32_t)q.size(-3) : 1;
    const int32_t m = (int32_t)q.size(-2), d = (int32_t)q.size(-1), n = (int32_t)k.size(-2);
    if ((int32_t)k.size(-1) != d || (int32_t)v.size(-1) != d || (int32_t)v.size(-2) != n ||
        (int32_t)o.size(-2) != m || (int32_t)o.size(-1) != d ||
        (rank == 3 && ((int32_t)o.size(-3) != heads || (int32_t)k.size(-3) != heads || (int32_t)v.size(-3) != heads)))
      throw std::logic_error("attention_f16: shape mismatch");
    auto z = [&](const TensorLayout& l) { return rank == 3 ? (int32_t)l.stride(-3) : 0; };
    auto call = [&](auto fn, auto... workspace) {
      return fn(stream_, o.ptr, q.ptr, k.ptr, v.ptr, heads, m, n, d,
                (int32_t)o.layout.stride(-1), (int32_t)o.layout.stride(-2), z(o.layout),
                (int32_t)q.layout.stride(-1), (int32_t)q.layout.stride(-2), z(q.layout),
                (int32_t)k.layout.stride(-1), (int32_t)k.layout.stride(-2), z(k.layout),
                (int32_t)v.layout.stride(-1), (int32_t)v.layout.stride(-2), z(v.layout),
                scale, temperature, (uint32_t)mask, workspace...);
    };
    int rc = workspace_bytes_ > 0 ? call(adr_attention_f16_ws, workspace_, workspace_bytes_) : call(adr_attention_f16);
    if (rc) throw AdrasteaError(rc, "attention_f16");
  }
  // kernels.rs:717-751: both operands flattened with shape_cast(&[-1]); equal lengths
  void error_stats_f16(TensorView<float>& out, const TensorView<const f16>& l, const TensorView<const f16>& r) override {
    auto lf = l.shape_cast({-1}), rf = r.shape_cast({-1});
    if (lf.size(-1) != rf.size(-1)) throw std::logic_error("error_stats: length mismatch");
    int rc = adr_error_stats_f16(stream_, descriptor(out), descriptor(lf), descriptor(rf));
    if (rc) throw AdrasteaError(rc, "error_stats_f16");
  }
  void error_stats_f32(TensorView<float>& out, const TensorView<const float>& l, const TensorView<const float>& r) override {
    auto lf = l.shape_cast({-1}), rf = r.shape_cast({-1});
    if (lf.size(-1) != rf.size(-1)) throw std::logic_error("error_stats: length mismatch");
    int rc = adr_error_stats_f32(stream_, descriptor(out), descriptor(lf), descriptor(rf));
    if (rc) throw AdrasteaError(rc, "error_stats_f32");
  }
  // A [heads, rows, d] view (rank 2: one head) as the C ABI takes it.
  struct Rows {
    int32_t heads, rows, d, x, y, z;
  };
  template <typename T>
  static Rows rows_of(const TensorView<T>& v, const char* what) {
    const auto& l = v.layout;
    if (l.dims.size() != 2 && l.dims.size() != 3) throw std::logic_error(std::string(what) + ": [heads, rows, d] views");
    const bool h = l.dims.size() == 3;
    auto size = [&](long i) { return int32_of(l.size(i), what); };
    auto stride = [&](long i) { return int32_of(l.stride(i), what, l.size(i) > 1); };
    return {h ? size(-3) : 1, size(-2), size(-1), stride(-1), stride(-2), h ? stride(-3) : 0};
  }
  static void same(const Rows& a, const Rows& b, const char* what) {
    if (a.heads != b.heads || a.rows != b.rows || a.d != b.d) throw std::logic_error(std::string(what) + ": shape mismatch");
  }
  void rotary_f16(TensorView<f16>& output, const TensorView<const f16>& input, const int32_t* positions,
                  const Rotary& rotary) override {
    const Rows o = rows_of(output, "rotary_f16"), i = rows_of(input, "rotary_f16");
    same(o, i, "rotary_f16");
    int rc = adr_rotary_f16(stream_, output.ptr, input.ptr, positions, rotary, i.heads, i.rows, i.d, o.x, o.y, o.z, i.x, i.y, i.z);
    if (rc) throw AdrasteaError(rc, "rotary_f16");
  }
  void append_f16(const PagedCache& cache, const PagedBatch& batch, const TensorView<const f16>& key, const TensorView<const f16>& value,
                  const Rotary& rotary, TensorView<f16>* query_out = nullptr, const TensorView<const f16>* query = nullptr,
                  const int32_t* positions = nullptr) override {
    const adr_paged_cache c = cache.lower();
    const Rows k = rows_of(key, "append_f16"), v = rows_of(value, "append_f16");
    same(k, v, "append_f16");
    if (k.heads != c.kv_heads || k.d != c.d || !query != !query_out) throw std::logic_error("append_f16: shape mismatch");
    Rows q{}, o{};
    if (query) {
      q = rows_of(*query, "append_f16"), o = rows_of(*query_out, "append_f16");
      same(q, o, "append_f16");
      if (q.rows != k.rows || q.d != k.d) throw std::logic_error("append_f16: shape mismatch");
    }
    int rc = adr_append_f16(stream_, c, batch, key.ptr, value.ptr, query ? query_out->ptr : nullptr, query ? query->ptr : nullptr,
                            positions, rotary, q.heads, k.rows, k.x, k.y, k.z, v.x, v.y, v.z, o.x, o.y, o.z, q.x, q.y, q.z);
    if (rc) throw AdrasteaError(rc, "append_f16");
  }
  void attention_paged_f16(TensorView<f16>& output, const TensorView<const f16>& query, const PagedCache& cache, const PagedBatch& batch,
                           float scale, float temperature = 1.0f, MatmulMask mask = MatmulMask::Causal) override {
    const adr_paged_cache c = cache.lower();
    const Rows o = rows_of(output, "attention_paged_f16"), q = rows_of(query, "attention_paged_f16");
    same(o, q, "attention_paged_f16");
    if (q.d != c.d) throw std::logic_error("attention_paged_f16: shape mismatch");
    auto call = [&](auto fn, auto... workspace) {
      return fn(stream_, output.ptr, query.ptr, c, batch, q.heads, q.rows, o.x, o.y, o.z, q.x, q.y, q.z, scale, temperature,
                (uint32_t)mask, workspace...);
    };
    int rc = workspace_bytes_ > 0 ? call(adr_attention_paged_f16_ws, workspace_, workspace_bytes_) : call(adr_attention_paged_f16);
    if (rc) throw AdrasteaError(rc, "attention_paged_f16");
  }
  void attention_packed_f16(TensorView<f16>& output, const TensorView<const f16>& query, const TensorView<const f16>& key,
                            const TensorView<const f16>& value, const PackedBatch& batch, float scale, float temperature = 1.0f,
                            MatmulMask mask = MatmulMask::Causal) override {
    const char* what = "attention_packed_f16";
    const Rows o = rows_of(output, what), q = rows_of(query, what), k = rows_of(key, what), v = rows_of(value, what);
    same(o, q, what), same(k, v, what);
    if (k.d != q.d) throw std::logic_error("attention_packed_f16: shape mismatch");
    auto call = [&](auto fn, auto... workspace) {
      return fn(stream_, output.ptr, query.ptr, key.ptr, value.ptr, batch, q.heads, k.heads, q.rows, k.rows, q.d, o.x, o.y, o.z, q.x,
                q.y, q.z, k.x, k.y, k.z, v.x, v.y, v.z, scale, temperature, (uint32_t)mask, workspace...);
    };
    int rc = workspace_bytes_ > 0 ? call(adr_attention_packed_f16_ws, workspace_, workspace_bytes_) : call(adr_attention_packed_f16);
    if (rc) throw AdrasteaError(rc, what);
  }
  void norm_rotary_f16(TensorView<f16>& output, const TensorView<const f16>& input, const int32_t* positions, int32_t pitch,
                       const RotaryAxes& rotary, const HeadNorm& norm) override {
    const Rows o = rows_of(output, "norm_rotary_f16"), i = rows_of(input, "norm_rotary_f16");
    same(o, i, "norm_rotary_f16");
    int rc = adr_norm_rotary_f16(stream_, output.ptr, input.ptr, positions, pitch, rotary, norm, i.heads, i.rows, i.d, o.x, o.y, o.z,
                                 i.x, i.y, i.z);
    if (rc) throw AdrasteaError(rc, "norm_rotary_f16");
  }
  void append_norm_f16(const PagedCache& cache, const PagedBatch& batch, const Appended& step) override {
    append(adr_append_norm_f16, "append_norm_f16", cache.lower(), batch, step);
  }
  void append_u8(const PagedCacheU8& cache, const PagedBatch& batch, const Appended& step) override {
    append(adr_append_u8, "append_u8", cache.lower(), batch, step);
  }
  void read_u8(TensorView<f16>& key_out, TensorView<f16>& value_out, const PagedCacheU8& cache, const PagedBatch& batch) override {
    const adr_paged_cache_u8 c = cache.lower();
    const Rows k = rows_of(key_out, "read_u8"), v = rows_of(value_out, "read_u8");
    same(k, v, "read_u8");
    if (k.heads != c.kv_heads || k.d != c.d) throw std::logic_error("read_u8: shape mismatch");
    int rc = adr_read_u8(stream_, key_out.ptr, value_out.ptr, c, batch, k.rows, k.x, k.y, k.z, v.x, v.y, v.z);
    if (rc) throw AdrasteaError(rc, "read_u8");
  }
  void attention_paged_u8(TensorView<f16>& output, const TensorView<const f16>& query, const PagedCacheU8& cache, const PagedBatch& batch,
                          float scale, float temperature = 1.0f, MatmulMask mask = MatmulMask::Causal) override {
    attend("attention_paged_u8", output, query, cache.lower(), [&](const Rows& o, const Rows& q, const adr_paged_cache_u8& c) {
      return workspace_bytes_ > 0 ? adr_attention_paged_u8_ws(stream_, output.ptr, query.ptr, c, batch, q.heads, q.rows, o.x, o.y, o.z, q.x,
                                                              q.y, q.z, scale, temperature, (uint32_t)mask, workspace_, workspace_bytes_)
                                  : adr_attention_paged_u8(stream_, output.ptr, query.ptr, c, batch, q.heads, q.rows, o.x, o.y, o.z, q.x,
                                                           q.y, q.z, scale, temperature, (uint32_t)mask);
    });
  }
  void attention_tree_f16(TensorView<f16>& output, const TensorView<const f16>& query, const PagedCache& cache, const PagedBatch& batch,
                          const DraftTree& tree, float scale, float temperature = 1.0f) override {
    attend("attention_tree_f16", output, query, cache.lower(), [&](const Rows& o, const Rows& q, const adr_paged_cache& c) {
      return workspace_bytes_ > 0 ? adr_attention_tree_f16_ws(stream_, output.ptr, query.ptr, c, batch, tree, q.heads, q.rows, o.x, o.y, o.z,
                                                              q.x, q.y, q.z, scale, temperature, workspace_, workspace_bytes_)
                                  : adr_attention_tree_f16(stream_, output.ptr, query.ptr, c, batch, tree, q.heads, q.rows, o.x, o.y, o.z,
                                                           q.x, q.y, q.z, scale, temperature);
    });
  }
  void attention_tree_u8(TensorView<f16>& output, const TensorView<const f16>& query, const PagedCacheU8& cache, const PagedBatch& batch,
                         const DraftTree& tree, float scale, float temperature = 1.0f) override {
    attend("attention_tree_u8", output, query, cache.lower(), [&](const Rows& o, const Rows& q, const adr_paged_cache_u8& c) {
      return workspace_bytes_ > 0 ? adr_attention_tree_u8_ws(stream_, output.ptr, query.ptr, c, batch, tree, q.heads, q.rows, o.x, o.y, o.z,
                                                             q.x, q.y, q.z, scale, temperature, workspace_, workspace_bytes_)
                                  : adr_attention_tree_u8(stream_, output.ptr, query.ptr, c, batch, tree, q.heads, q.rows, o.x, o.y, o.z,
                                                          q.x, q.y, q.z, scale, temperature);
    });
  }
  std::string plan(const TensorLayout& o, const TensorLayout& l, const TensorLayout& r, const MatmulOptions& opt) const {
    LoweredMatmul w = lower_matmul(o, l, r, opt);
    char name[64];
    int rc = adr_matmul_f16_plan(name, sizeof name, w.batches, w.m, w.k, w.n, w.so[0], w.so[1], w.so[2], w.sl[0],
                                 w.sl[1], w.sl[2], w.sr[0], w.sr[1], w.sr[2], w.store, w.load, w.mask);
    if (rc) throw AdrasteaError(rc, "matmul_f16_plan");
    return name;
  }

 private:
  template <typename F>
  void run(F fn, const char* what, TensorView<f16>& o, const TensorView<const f16>& l,
           const TensorView<const f16>& r, const MatmulOptions& opt) {
    LoweredMatmul w = lower_matmul(o.layout, l.layout, r.layout, opt);
    int rc = fn(stream_, o.ptr, l.ptr, r.ptr, w.batches, w.m, w.k, w.n, w.so[0], w.so[1], w.so[2], w.sl[0], w.sl[1],
                w.sl[2], w.sr[0], w.sr[1], w.sr[2], opt.store_.bias, w.beta, w.scale, w.store, w.load, w.mask);
    if (rc) throw AdrasteaError(rc, what);
  }
  template <typename F, typename Cache>
  void append(F fn, const char* what, const Cache& c, const PagedBatch& batch, const Appended& step) {
    const Rows k = rows_of(step.key, what), v = rows_of(step.value, what);
    same(k, v, what);
    if (k.heads != c.kv_heads || k.d != c.d || !step.query != !step.query_out) throw std::logic_error(std::string(what) + ": shape mismatch");
    Rows q{}, o{};
    if (step.query) {
      q = rows_of(*step.query, what), o = rows_of(*step.query_out, what);
      same(q, o, what);
      if (q.rows != k.rows || q.d != k.d) throw std::logic_error(std::string(what) + ": shape mismatch");
    }
    int rc = fn(stream_, c, batch, step.key.ptr, step.value.ptr, step.query ? step.query_out->ptr : nullptr,
                step.query ? step.query->ptr : nullptr, step.positions, step.pitch, step.rotary, step.query_norm, step.key_norm, q.heads,
                k.rows, k.x, k.y, k.z, v.x, v.y, v.z, o.x, o.y, o.z, q.x, q.y, q.z);
    if (rc) throw AdrasteaError(rc, what);
  }
  template <typename Cache, typename F>
  void attend(const char* what, const TensorView<f16>& output, const TensorView<const f16>& query, const Cache& c, F call) {
    const Rows o = rows_of(output, what), q = rows_of(query, what);
    same(o, q, what);
    if (q.d != c.d) throw std::logic_error(std::string(what) + ": shape mismatch");
    int rc = call(o, q, c);
    if (rc) throw AdrasteaError(rc, what);
  }
  adr_stream_t stream_;
  void* workspace_;
  int64_t workspace_bytes_;
};

// Records the set of (left, right, output) layouts seen, then forwards (kernels.rs:231-359).
class MatmulTracer : public CommonKernels {
 public:
  explicit MatmulTracer(CommonKernels& inner) : inner_(inner) {}
  void clear() { std::lock_guard<std::mutex> g(mu_); shapes_.clear(); }
  std::set<std::tuple<TensorLayout, TensorLayout, TensorLayout>> shapes() { std::lock_guard<std::mutex> g(mu_); return shapes_; }
  void matmul_f16(TensorView<f16>& o, const TensorView<const f16>& l, const TensorView<const f16>& r,
                  const MatmulOptions& opt) override { rec(o, l, r); inner_.matmul_f16(o, l, r, opt); }
  void matmul_f16_slow(TensorView<f16>& o, const TensorView<const f16>& l, const TensorView<const f16>& r,
                       const MatmulOptions& opt) override { rec(o, l, r); inner_.matmul_f16_slow(o, l, r, opt); }
  void softmax_rows_inplace(TensorView<f16>& o, float t) override { inner_.softmax_rows_inplace(o, t); }
  void attention_f16(TensorView<f16>& o, const TensorView<const f16>& q, const TensorView<const f16>& k,
                     const TensorView<const f16>& v, float scale, float t, MatmulMask mask) override {
    inner_.attention_f16(o, q, k, v, scale, t, mask);
  }
  void error_stats_f16(TensorView<float>& out, const TensorView<const f16>& l, const TensorView<const f16>& r) override { inner_.error_stats_f16(out, l, r); }
  void error_stats_f32(TensorView<float>& out, const TensorView<const float>& l, const TensorView<const float>& r) override { inner_.error_stats_f32(out, l, r); }
  void rotary_f16(TensorView<f16>& o, const TensorView<const f16>& i, const int32_t* positions, const Rotary& rotary) override {
    inner_.rotary_f16(o, i, positions, rotary);
  }
  void append_f16(const PagedCache& cache, const PagedBatch& batch, const TensorView<const f16>& k, const TensorView<const f16>& v,
                  const Rotary& rotary, TensorView<f16>* query_out = nullptr, const TensorView<const f16>* query = nullptr,
                  const int32_t* positions = nullptr) override {
    inner_.append_f16(cache, batch, k, v, rotary, query_out, query, positions);
  }
  void attention_paged_f16(TensorView<f16>& o, const TensorView<const f16>& q, const PagedCache& cache, const PagedBatch& batch,
                           float scale, float t = 1.0f, MatmulMask mask = MatmulMask::Causal) override {
    inner_.attention_paged_f16(o, q, cache, batch, scale, t, mask);
  }
  void attention_packed_f16(TensorView<f16>& o, const TensorView<const f16>& q, const TensorView<const f16>& k,
                            const TensorView<const f16>& v, const PackedBatch& batch, float scale, float t = 1.0f,
                            MatmulMask mask = MatmulMask::Causal) override {
    inner_.attention_packed_f16(o, q, k, v, batch, scale, t, mask);
  }
  void norm_rotary_f16(TensorView<f16>& o, const TensorView<const f16>& i, const int32_t* positions, int32_t pitch, const RotaryAxes& rotary,
                       const HeadNorm& norm) override {
    inner_.norm_rotary_f16(o, i, positions, pitch, rotary, norm);
  }
  void append_norm_f16(const PagedCache& cache, const PagedBatch& batch, const Appended& step) override { inner_.append_norm_f16(cache, batch, step); }
  void append_u8(const PagedCacheU8& cache, const PagedBatch& batch, const Appended& step) override { inner_.append_u8(cache, batch, step); }
  void read_u8(TensorView<f16>& k, TensorView<f16>& v, const PagedCacheU8& cache, const PagedBatch& batch) override { inner_.read_u8(k, v, cache, batch); }
  void attention_paged_u8(TensorView<f16>& o, const TensorView<const f16>& q, const PagedCacheU8& cache, const PagedBatch& batch,
                          float scale, float t = 1.0f, MatmulMask mask = MatmulMask::Causal) override {
    inner_.attention_paged_u8(o, q, cache, batch, scale, t, mask);
  }
  void attention_tree_f16(TensorView<f16>& o, const TensorView<const f16>& q, const PagedCache& cache, const PagedBatch& batch,
                          const DraftTree& tree, float scale, float t = 1.0f) override {
    inner_.attention_tree_f16(o, q, cache, batch, tree, scale, t);
  }
  void attention_tree_u8(TensorView<f16>& o, const TensorView<const f16>& q, const PagedCacheU8& cache, const PagedBatch& batch,
                         const DraftTree& tree, float scale, float t = 1.0f) override {
    inner_.attention_tree_u8(o, q, cache, batch, tree, scale, t);
  }

 private:
  void rec(const TensorView<f16>& o, const TensorView<const f16>& l, const TensorView<const f16>& r) {
    std::lock_guard<std::mutex> g(mu_);
    shapes_.insert(std::make_tuple(l.layout, r.layout, o.layout));
  }
  CommonKernels& inner_;
  std::mutex mu_;
  std::set<std::tuple<TensorLayout, TensorLayout, TensorLayout>> shapes_;
};

}  // namespace adrastea
