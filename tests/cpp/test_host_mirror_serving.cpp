// The serving calls of the C++ host mirror (include/molten_b200.hpp) without a
// GPU: their checks throw before the C ABI is reached, and a well-formed call
// reaches it (a null context, which the ABI rejects with its own message).
#include <cstdio>
#include <cstring>

#include "molten_b200.hpp"

using molten::DType;
using molten::Error;
using molten::Tensor;
namespace kernels = molten::kernels;

static int failures = 0;

template <typename F>
static void expect_error(const char* what, const char* needle, F&& f) {
  try {
    f();
    std::printf("FAIL %s: no error\n", what);
    ++failures;
  } catch (const Error& e) {
    if (std::strstr(e.what(), needle) == nullptr) {
      std::printf("FAIL %s: message '%s'\n", what, e.what());
      ++failures;
    }
  }
}

int main() {
  // never dereferenced; apart, so that nothing overlaps
  uintptr_t at = 0x1000000;
  auto T = [&](std::initializer_list<int64_t> s, DType d) {
    Tensor t(reinterpret_cast<void*>(at), s, d);
    at += 0x1000000;
    return t;
  };
  molten::Context ctx = molten::Context::wrap(nullptr);
  const Tensor lens = T({4}, DType::U32), table = T({4, 8}, DType::U32), free = T({32}, DType::U32);
  const Tensor one = T({1}, DType::U32), start = T({5}, DType::U32), map = T({4}, DType::U32);
  const Tensor slots = T({4}, DType::U64);
  expect_error("plan reaches the ABI", "null context", [&] {
    kernels::kv_plan(ctx, lens, nullptr, 16, table, free, one, lens, one, start, map, map, map, slots);
  });
  expect_error("plan row_start", "row_start shape", [&] {
    kernels::kv_plan(ctx, lens, nullptr, 16, table, free, one, lens, one, lens, map, map, map, slots);
  });
  expect_error("release reaches the ABI", "null context",
               [&] { kernels::kv_release(ctx, lens, lens, 16, table, free, one, lens, one); });
  expect_error("release done", "done shape",
               [&] { kernels::kv_release(ctx, one, lens, 16, table, free, one, lens, one); });

  kernels::KvCache cache{T({32, 8, 16, 64}, DType::BF16), T({32, 8, 16, 64}, DType::BF16)};
  const Tensor q = T({4, 32, 64}, DType::BF16), k = T({4, 8, 64}, DType::BF16);
  const Tensor v = T({4, 8, 64}, DType::BF16), out = T({4, 32, 64}, DType::BF16);
  const Tensor gain = T({64}, DType::BF16), turns = T({32}, DType::U64);
  expect_error("rope reaches the ABI", "null context", [&] {
    kernels::qk_norm_rope(ctx, q, 0, k, 0, &v, 0, &gain, &gain, 1e-5f, &map, &turns, false, out, 0,
                          cache, &slots);
  });
  expect_error("rope k rows", "match the cache", [&] {
    kernels::qk_norm_rope(ctx, q, 0, q, 0, &v, 0, &gain, &gain, 1e-5f, &map, &turns, false, out, 0,
                          cache, &slots);
  });
  expect_error("rope without positions", "turns", [&] {
    kernels::qk_norm_rope(ctx, q, 0, k, 0, &v, 0, &gain, &gain, 1e-5f, nullptr, &turns, false, out,
                          0, cache, &slots);
  });
  const Tensor ws = T({1 << 22}, DType::U32), lse = T({4, 32}, DType::F32);
  expect_error("attention reaches the ABI", "null context", [&] {
    kernels::paged_attention(ctx, q, cache, table, map, nullptr, 0, 0.125f, out, &lse, ws);
  });
  expect_error("attention workspace", "workspace", [&] {
    kernels::paged_attention(ctx, q, cache, table, map, nullptr, 0, 0.125f, out, &lse, one);
  });
  expect_error("attention heads", "query heads", [&] {
    const Tensor q9 = T({4, 9, 64}, DType::BF16);
    kernels::paged_attention(ctx, q9, cache, table, map, nullptr, 0, 0.125f, q9, nullptr, ws);
  });
  kernels::KvCache bad = cache;
  bad.v.dtype = DType::E4M3;
  expect_error("unlike caches", "alike", [&] {
    kernels::paged_attention(ctx, q, bad, table, map, nullptr, 0, 0.125f, out, &lse, ws);
  });

  bad = cache;
  bad.k = bad.v = T({8, 0, 16, 64}, DType::BF16);
  expect_error("empty cache", "empty", [&] {
    kernels::paged_attention(ctx, q, bad, table, map, nullptr, 0, 0.125f, out, &lse, ws);
  });
  const Tensor wide = T({64}, DType::F32);
  expect_error("gains of another type", "gains", [&] {
    kernels::qk_norm_rope(ctx, q, 0, k, 0, &v, 0, &wide, &gain, 1e-5f, &map, &turns, false, out, 0,
                          cache, &slots);
  });

  const Tensor logits = T({2, 1000}, DType::BF16), to = T({2, 1000}, DType::BF16);
  const Tensor seen = T({2, 32}, DType::U32), counts = T({2, 1000}, DType::U16);
  const Tensor f = T({2}, DType::F32), best = T({2}, DType::U64), toks = T({2}, DType::U32);
  kernels::LogitsRules r;
  r.seen = &seen;
  r.repetition = &f;
  r.counts = &counts;
  r.frequency = &f;
  expect_error("rules reach the ABI", "null context",
               [&] { kernels::logits_process(ctx, logits, to, r, &best); });
  expect_error("mark reaches the ABI", "null context",
               [&] { kernels::logits_mark(ctx, toks, r, 1000); });
  expect_error("mark of another vocabulary", "seen shape",
               [&] { kernels::logits_mark(ctx, toks, r, 2000); });
  r.seen = &counts;
  expect_error("rules seen", "seen shape", [&] { kernels::logits_process(ctx, logits, to, r); });
  r.seen = nullptr;
  expect_error("rules seen without", "go together",
               [&] { kernels::logits_process(ctx, logits, to, r); });
  std::printf("%s (%d failures)\n", failures ? "FAILED" : "ok", failures);
  return failures != 0;
}
