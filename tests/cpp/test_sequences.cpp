// The calls over several sequences through the C++ host mirror.  Without arguments: what is refused on the host, and the
// lowering of a cache.  With "gpu": a step of two sequences -- keys and values to their pages, attention over
// them -- with values that make every result exact.
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

static void cpu_tests() {
  const PagedCache cache{{P, TensorLayout::row_major({6, 16, 2, 64}).permute({0, 2, 1, 3})},
                         {P + 8, TensorLayout::row_major({6, 2, 16, 64})}};
  const adr_paged_cache c = cache.lower();
  CHECK(c.key == P && c.value == P + 8 && c.pages == 6 && c.kv_heads == 2 && c.page_size == 16 && c.d == 64);
  CHECK(c.stride_kx == 1 && c.stride_ky == 128 && c.stride_kz == 64 && c.stride_kp == 2048);
  CHECK(c.stride_vx == 1 && c.stride_vy == 64 && c.stride_vz == 1024 && c.stride_vp == 2048);
  CHECK(throws([&] { PagedCache{cache.key, {P, TensorLayout::row_major({5, 2, 16, 64})}}.lower(); }));
  CHECK(throws([&] { PagedCache{{P, TensorLayout::row_major({6, 2, 64})}, {P, TensorLayout::row_major({6, 2, 64})}}.lower(); }));

  GpuKernels gpu;
  MatmulTracer k(gpu);  // (forwards them)
  const PagedBatch batch{(const int32_t*)P, (const int32_t*)P, (const int32_t*)P, 2, 3, 3, 1, 48};
  TensorView<f16> out(P, TensorLayout::row_major({4, 3, 64})), fewer(P, TensorLayout::row_major({4, 2, 64}));
  const TensorView<const f16> q(P, out.layout), kv(P, TensorLayout::row_major({2, 3, 64})), wide(P, TensorLayout::row_major({4, 3, 72}));
  const Rotary none{nullptr, 0, ADR_ROTARY_HALVES, 1.0f};
  CHECK(throws([&] { k.attention_paged_f16(fewer, q, cache, batch, 0.1f); }));
  CHECK(throws([&] { TensorView<f16> w(P, wide.layout); k.attention_paged_f16(w, wide, cache, batch, 0.1f); }));
  CHECK(throws([&] { k.append_f16(cache, batch, q, q, none); }));                       // four heads, the cache has two
  CHECK(throws([&] { k.append_f16(cache, batch, kv, kv, none, &out, nullptr); }));      // a result without queries
  CHECK(throws([&] { k.rotary_f16(fewer, q, (const int32_t*)P, none); }));
  CHECK(throws([&] { k.attention_packed_f16(out, q, kv, wide, PackedBatch{}, 0.1f); }));
  try {
    k.attention_paged_f16(out, q, cache, batch, -1.0f);
    CHECK(false);
  } catch (const AdrasteaError& e) {
    CHECK(e.code == ADR_EUNSUPPORTED_LAYOUT);
  }
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
  int refused = 0;
  auto code = [&](auto call) {
    try { call(); } catch (const AdrasteaError& e) { refused += e.code == ADR_ENOTIMPL; }
  };
  code([&] { over_other.rotary_f16(out, q, (const int32_t*)P, none); });
  code([&] { over_other.append_f16(cache, batch, kv, kv, none); });
  code([&] { over_other.attention_paged_f16(out, q, cache, batch, 0.1f); });
  code([&] { over_other.attention_packed_f16(out, q, kv, kv, PackedBatch{}, 0.1f); });
  CHECK(refused == 4);
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
  // Two sequences with 17 and 3 keys, of which 2 and 1 are new; keys all zero, so that every key weighs the same, and
  // value rows that hold 1 for the first sequence's new keys, 0 for its old ones, 3 everywhere in the second.
  const int heads = 4, kv = 2, d = 64, page = 16, pages = 4, rows = 3;
  const uint16_t one = 0x3c00, three = 0x4200;
  std::vector<f16> pool_k(pages * kv * page * d, 0), pool_v(pool_k.size(), 0), q(rows * heads * d, one), k(rows * kv * d, 0), v(k.size());
  for (int r = 0; r < rows; r++)
    for (int i = 0; i < kv * d; i++) v[r * kv * d + i] = r < 2 ? one : three;
  const std::vector<int32_t> offsets{0, 2, 3}, lengths{17, 3}, table{2, 0, 3, -1};
  for (int s = 0; s < 2; s++)  // (the second sequence's old values)
    for (int h = 0; h < kv; h++)
      for (int i = 0; i < d; i++) pool_v[((3 * kv + h) * page + s) * d + i] = three;
  const auto cache_layout = TensorLayout::row_major({(size_t)pages, (size_t)kv, (size_t)page, (size_t)d});
  const PagedCache cache{{(f16*)put(pool_k.data(), pool_k.size() * 2), cache_layout}, {(f16*)put(pool_v.data(), pool_v.size() * 2), cache_layout}};
  const PagedBatch batch{(const int32_t*)put(offsets.data(), 12), (const int32_t*)put(lengths.data(), 8),
                         (const int32_t*)put(table.data(), 16), 2, 2, 2, 2, 17};
  auto view = [&](int h) { return TensorLayout::row_major({(size_t)rows, (size_t)h, (size_t)d}).permute({1, 0, 2}); };
  TensorView<f16> out((f16*)put(q.data(), q.size() * 2), view(heads));
  const TensorView<const f16> qv((const f16*)put(q.data(), q.size() * 2), view(heads)), kview((const f16*)put(k.data(), k.size() * 2), view(kv)),
      vview((const f16*)put(v.data(), v.size() * 2), view(kv));
  GpuKernels gpu;
  MatmulTracer kernels(gpu);
  kernels.append_f16(cache, batch, kview, vview, Rotary{nullptr, 0, ADR_ROTARY_HALVES, 1.0f});
  kernels.attention_paged_f16(out, qv, cache, batch, 0.125f);
  CHECK(sync() == 0);
  std::vector<f16> got(q.size());
  CHECK(copy(got.data(), out.ptr, got.size() * 2, 2) == 0);
  // 1/16 of keys that weigh the same is exact; 2/17 is fp16's neighbour of it, and its probability sum's
  for (int i = 0; i < heads * d; i++) {
    CHECK(got[i] == 0x2c00);                                                             // 1/16
    CHECK(got[heads * d + i] >= 0x2f87 && got[heads * d + i] <= 0x2f88);                 // 2/17 = 0.117647
    CHECK(got[2 * heads * d + i] == three);
  }
  // packed: each row sees itself and what is before it
  const PackedBatch packed{batch.row_offsets, batch.row_offsets, 2, 2, 2};
  kernels.attention_packed_f16(out, qv, kview, vview, packed, 0.125f);
  CHECK(sync() == 0 && copy(got.data(), out.ptr, got.size() * 2, 2) == 0);
  for (int i = 0; i < heads * d; i++) CHECK(got[i] == one && got[heads * d + i] == one && got[2 * heads * d + i] == three);
  // a quarter turn at position 1: (1, 1) -> (-1, 1)
  const double quarter[32] = {0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25,
                              0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25, 0.25};
  const std::vector<int32_t> positions{0, 1, 2};
  kernels.rotary_f16(out, qv, (const int32_t*)put(positions.data(), 12), Rotary{(const double*)put(quarter, 256), 64, ADR_ROTARY_HALVES, 1.0f});
  CHECK(sync() == 0 && copy(got.data(), out.ptr, got.size() * 2, 2) == 0);
  for (int h = 0; h < heads; h++)
    for (int i = 0; i < d; i++) {
      const uint16_t minus = 0xbc00, a = got[h * d + i], b = got[(heads + h) * d + i], c = got[(2 * heads + h) * d + i];
      CHECK(a == one && b == (i < 32 ? minus : one) && c == minus);
    }
}

int main(int argc, char** argv) {
  if (argc > 1 && !strcmp(argv[1], "gpu")) gpu_tests();
  else cpu_tests();
  if (!failures) printf("OK\n");
  return failures != 0;
}
