// Heads normed and turned, a cache in 8 bits and drafted trees through the C++ host mirror.  Without arguments: what is refused on
// the host, and the lowering of a cache of codes.  With "gpu": steps of two sequences with values that make every result exact, or
// known to a rounding.
#include <dlfcn.h>

#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "../../adrastea_amd/host/kernels.hpp"

using namespace adrastea;

static int failures = 0;
#define CHECK(c) do { if (!(c)) { printf("FAIL %s:%d %s\n", __FILE__, __LINE__, #c); failures++; } } while (0)
template <typename F> static bool throws(F f) { try { f(); } catch (const std::exception&) { return true; } return false; }

static f16* const P = (f16*)4096;  // never read

static PagedCacheU8 codes(uint8_t* k, f16* ks, uint8_t* v, f16* vs, size_t pages, size_t heads, size_t page, size_t d) {
  return {{k, TensorLayout::row_major({pages, page, heads, d}).permute({0, 2, 1, 3})}, {ks, TensorLayout::row_major({pages, heads, page})},
          {v, TensorLayout::row_major({pages, heads, page, d})}, {vs, TensorLayout::row_major({pages, page, heads}).permute({0, 2, 1})}};
}

static void cpu_tests() {
  const PagedCacheU8 cache = codes((uint8_t*)P, P + 1, (uint8_t*)(P + 2), P + 3, 6, 2, 16, 64);
  const adr_paged_cache_u8 c = cache.lower();
  CHECK(c.key == (uint8_t*)P && c.key_scale == P + 1 && c.value == (uint8_t*)(P + 2) && c.value_scale == P + 3);
  CHECK(c.pages == 6 && c.kv_heads == 2 && c.page_size == 16 && c.d == 64);
  CHECK(c.stride_kx == 1 && c.stride_ky == 128 && c.stride_kz == 64 && c.stride_kp == 2048);
  CHECK(c.stride_vx == 1 && c.stride_vy == 64 && c.stride_vz == 1024 && c.stride_vp == 2048);
  CHECK(c.stride_ksy == 1 && c.stride_ksz == 16 && c.stride_ksp == 32 && c.stride_vsy == 2 && c.stride_vsz == 1 && c.stride_vsp == 32);
  CHECK(throws([&] { PagedCacheU8 other = cache; other.value = {(uint8_t*)P, TensorLayout::row_major({5, 2, 16, 64})}; other.lower(); }));
  CHECK(throws([&] { PagedCacheU8 other = cache; other.key_scale = {P, TensorLayout::row_major({6, 2, 15})}; other.lower(); }));
  CHECK(throws([&] { PagedCacheU8 other = cache; other.value_scale = {P, TensorLayout::row_major({6, 2, 16, 1})}; other.lower(); }));

  GpuKernels gpu;
  MatmulTracer k(gpu);  // (forwards them)
  const PagedBatch batch{(const int32_t*)P, (const int32_t*)P, (const int32_t*)P, 2, 3, 3, 1, 48};
  TensorView<f16> out(P, TensorLayout::row_major({4, 3, 64})), fewer(P, TensorLayout::row_major({4, 2, 64})), kv_out(P, TensorLayout::row_major({2, 3, 64}));
  const TensorView<const f16> q(P, out.layout), kv(P, kv_out.layout), wide(P, TensorLayout::row_major({4, 3, 72}));
  const PagedCache halves{{P, TensorLayout::row_major({6, 2, 16, 64})}, {P, TensorLayout::row_major({6, 2, 16, 64})}};
  const RotaryAxes none{nullptr, nullptr, 0, ADR_ROTARY_HALVES, 1.0f, 1};
  const DraftTree tree{(const int32_t*)P, 1, 1};
  CHECK(throws([&] { k.norm_rotary_f16(fewer, q, nullptr, 0, none, HeadNorm{}); }));
  CHECK(throws([&] { k.append_norm_f16(halves, batch, Appended{q, q}); }));  // four heads, the cache has two
  CHECK(throws([&] { Appended a{kv, kv}; a.query_out = &out; k.append_u8(cache, batch, a); }));  // a result without queries
  CHECK(throws([&] { Appended a{kv, kv}; a.query_out = &fewer, a.query = &q; k.append_u8(cache, batch, a); }));
  CHECK(throws([&] { k.read_u8(kv_out, out, cache, batch); }));
  CHECK(throws([&] { k.read_u8(out, out, cache, batch); }));
  CHECK(throws([&] { k.attention_paged_u8(fewer, q, cache, batch, 0.1f); }));
  CHECK(throws([&] { TensorView<f16> w(P, wide.layout); k.attention_tree_f16(w, wide, halves, batch, tree, 0.1f); }));
  CHECK(throws([&] { TensorView<f16> w(P, wide.layout); k.attention_tree_u8(w, wide, cache, batch, tree, 0.1f); }));
  auto refused_with = [&](int code, auto call) {
    try { call(); } catch (const AdrasteaError& e) { return e.code == code; }
    return false;
  };
  CHECK(refused_with(ADR_EUNSUPPORTED_LAYOUT, [&] { k.attention_paged_u8(out, q, cache, batch, -1.0f); }));
  CHECK(refused_with(ADR_EUNSUPPORTED_LAYOUT, [&] { k.attention_tree_u8(out, q, cache, batch, tree, -1.0f); }));
  CHECK(refused_with(ADR_EINVAL_SHAPE, [&] { k.norm_rotary_f16(out, q, nullptr, 0, none, HeadNorm{P, -1.0f}); }));
  struct Other : CommonKernels {  // an implementation from before these calls
    void matmul_f16(TensorView<f16>&, const TensorView<const f16>&, const TensorView<const f16>&, const MatmulOptions&) override {}
    void matmul_f16_slow(TensorView<f16>&, const TensorView<const f16>&, const TensorView<const f16>&, const MatmulOptions&) override {}
    void softmax_rows_inplace(TensorView<f16>&, float) override {}
    void attention_f16(TensorView<f16>&, const TensorView<const f16>&, const TensorView<const f16>&, const TensorView<const f16>&, float,
                       float, MatmulMask) override {}
    void error_stats_f16(TensorView<float>&, const TensorView<const f16>&, const TensorView<const f16>&) override {}
    void error_stats_f32(TensorView<float>&, const TensorView<const float>&, const TensorView<const float>&) override {}
  } other;
  MatmulTracer over_other(other);
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.norm_rotary_f16(out, q, nullptr, 0, none, HeadNorm{}); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.append_norm_f16(halves, batch, Appended{kv, kv}); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.append_u8(cache, batch, Appended{kv, kv}); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.read_u8(kv_out, kv_out, cache, batch); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.attention_paged_u8(out, q, cache, batch, 0.1f); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.attention_tree_f16(out, q, halves, batch, tree, 0.1f); }));
  CHECK(refused_with(ADR_ENOTIMPL, [&] { over_other.attention_tree_u8(out, q, cache, batch, tree, 0.1f); }));
}

static void gpu_tests() {
  void* hip = dlopen("libamdhip64.so", RTLD_NOW | RTLD_GLOBAL);
  if (!hip) { printf("FAIL no HIP runtime\n"); failures++; return; }
  auto alloc = (int (*)(void**, size_t))dlsym(hip, "hipMalloc");
  auto copy = (int (*)(void*, const void*, size_t, int))dlsym(hip, "hipMemcpy");
  auto sync = (int (*)())dlsym(hip, "hipDeviceSynchronize");
  auto put = [&](const void* p, size_t n) {
    void* d = nullptr;
    CHECK(alloc(&d, n) == 0 && copy(d, p, n, 1) == 0);
    return d;
  };
  auto get = [&](const void* d, size_t n) {
    std::vector<f16> got(n);
    CHECK(sync() == 0 && copy(got.data(), d, n * 2, 2) == 0);
    return got;
  };
  // Two sequences of 17 and 3 keys, all of them appended: 16 + 2 rows, then drafts of 1 + 1.  Keys are zeros, so that every key
  // weighs the same; a value is 1 or 3 everywhere (scale 1 / 127.5 up, codes 255).
  const int heads = 4, kv = 2, d = 64, page = 16, pages = 4;
  const uint16_t one = 0x3c00, three = 0x4200;
  const size_t slots = (size_t)pages * kv * page;
  const std::vector<f16> zeros(slots * d, 0), ones(18 * heads * d, one);
  std::vector<f16> v(18 * kv * d);
  for (size_t i = 0; i < v.size(); i++) v[i] = (int)i < 16 * kv * d ? one : three;
  const std::vector<int32_t> table{2, 0, 3, -1}, offsets{0, 16, 18}, lengths{16, 2}, offsets2{0, 1, 2}, lengths2{17, 3};
  const PagedCacheU8 cache = codes((uint8_t*)put(zeros.data(), slots * d), (f16*)put(zeros.data(), slots * 2),
                                   (uint8_t*)put(zeros.data(), slots * d), (f16*)put(zeros.data(), slots * 2), pages, kv, page, d);
  const int32_t* const where = (const int32_t*)put(table.data(), 16);
  const PagedBatch prompts{(const int32_t*)put(offsets.data(), 12), (const int32_t*)put(lengths.data(), 8), where, 2, 2, 2, 16, 16};
  const PagedBatch drafts{(const int32_t*)put(offsets2.data(), 12), (const int32_t*)put(lengths2.data(), 8), where, 2, 2, 2, 1, 17};
  auto view = [&](int rows, int h) { return TensorLayout::row_major({(size_t)rows, (size_t)h, (size_t)d}).permute({1, 0, 2}); };
  const f16* const k_at = (const f16*)put(zeros.data(), v.size() * 2);
  const f16* const v_at = (const f16*)put(v.data(), v.size() * 2);
  const f16* const q_at = (const f16*)put(ones.data(), ones.size() * 2);
  f16* const out_at = (f16*)put(ones.data(), ones.size() * 2);
  GpuKernels gpu;
  MatmulTracer kernels(gpu);
  kernels.append_u8(cache, prompts, Appended{{k_at, view(18, kv)}, {v_at, view(18, kv)}});
  // (the drafts: a one for the first sequence, a three for the second)
  kernels.append_u8(cache, drafts, Appended{{k_at, view(2, kv)}, {v_at + 15 * kv * d, view(2, kv)}});
  TensorView<f16> out(out_at, view(2, heads)), back_k(out_at, view(18, kv)), back_v(out_at + 18 * kv * d, view(18, kv));
  const TensorView<const f16> q(q_at, view(2, heads));
  kernels.read_u8(back_k, back_v, cache, prompts);
  std::vector<f16> got = get(out_at, 2 * 18 * kv * d);
  for (int i = 0; i < 18 * kv * d; i++) {
    CHECK(got[i] == 0);
    // (the scale is at most 2^-10 above top / 127.5; half a scale of 255 is 2^-9: next to the value)
    const uint16_t want = i < 16 * kv * d ? one : three;
    CHECK(got[18 * kv * d + i] >= want - 4 && got[18 * kv * d + i] <= want + 2);
  }
  // Every key weighs the same: 16 ones and a one (the row in front of the second's), 2 threes and a three
  kernels.attention_paged_u8(out, q, cache, drafts, 0.125f);
  got = get(out_at, 2 * heads * d);
  for (int i = 0; i < heads * d; i++) {
    CHECK(got[i] >= one - 4 && got[i] <= one + 2);
    CHECK(got[heads * d + i] >= three - 4 && got[heads * d + i] <= three + 2);
  }
  // A draft whose rows see no drafted key, not themselves either: only what is in front
  const std::vector<int32_t> nothing{0, 0};
  const DraftTree tree{(const int32_t*)put(nothing.data(), 8), 1, 1};
  kernels.attention_tree_u8(out, q, cache, drafts, tree, 0.125f);
  got = get(out_at, 2 * heads * d);
  for (int i = 0; i < heads * d; i++) {
    CHECK(got[i] >= one - 4 && got[i] <= one + 2);
    CHECK(got[heads * d + i] >= three - 4 && got[heads * d + i] <= three + 2);
  }
  // The same in 16 bits, through append_norm_f16: the values are exact, so their means are
  const auto cache_layout = TensorLayout::row_major({(size_t)pages, (size_t)kv, (size_t)page, (size_t)d});
  const PagedCache halves{{(f16*)put(zeros.data(), slots * d * 2), cache_layout}, {(f16*)put(zeros.data(), slots * d * 2), cache_layout}};
  kernels.append_norm_f16(halves, prompts, Appended{{k_at, view(18, kv)}, {v_at, view(18, kv)}});
  kernels.append_norm_f16(halves, drafts, Appended{{k_at, view(2, kv)}, {v_at + 15 * kv * d, view(2, kv)}});
  kernels.attention_tree_f16(out, q, halves, drafts, tree, 0.125f);
  got = get(out_at, 2 * heads * d);
  for (int i = 0; i < heads * d; i++) CHECK(got[i] == one && got[heads * d + i] == three);
  // A norm and two axes: heads of ones stay ones; half of the pairs turned by a quarter on the second axis, (1, 1) -> (-1, 1)
  std::vector<double> quarter(32, 0.25);
  std::vector<int32_t> axis(32), positions{0, 0, 5, 1, 0, 5};  // [2][3], of which two rows are used
  for (int i = 0; i < 32; i++) axis[i] = i & 1;
  kernels.norm_rotary_f16(out, q, (const int32_t*)put(positions.data(), 24), 3,
                          RotaryAxes{(const double*)put(quarter.data(), 256), (const int32_t*)put(axis.data(), 128), d, ADR_ROTARY_HALVES, 1.0f, 2},
                          HeadNorm{q_at, 0.0f});
  got = get(out_at, 2 * heads * d);
  for (int i = 0; i < heads * d; i++) {
    const uint16_t minus = 0xbc00;
    CHECK(got[i] == ((i % d) < 32 && (i & 1) ? minus : one) && got[heads * d + i] == one);
  }
}

int main(int argc, char** argv) {
  if (argc > 1 && !strcmp(argv[1], "gpu")) gpu_tests();
  else cpu_tests();
  if (!failures) printf("OK\n");
  return failures != 0;
}
