// A request's rules on its logits, for a batch of rows, before the draw
// (mc_logits_process), and the counts they go by (mc_logits_mark).
//
// For token i of row b, in fp32 and in this order:
//   seen:     v = v > 0 ? v / rep_b : v * rep_b
//   counts:   v = v - freq_b * count_i - (count_i > 0 ? pres_b : 0)
//   biases:   v = v + sum of the row's biases for i (in list order)
//   grammar:  v = -inf where the bitmap leaves i out, whatever v was
// rounded once to the logits' type; the stored value also goes into the
// 64-bit greedy key of the head (largest value, ties to the lowest id, NaN
// never), which mc_token_tail reads.
//
// What bounds it: bytes, 2 to 8 read and 2 or 4 written a token. A thread
// takes 8 tokens: one 16-byte load of bf16 logits, one of counts, one byte of
// each bitmap. A CTA takes 2048 tokens of one row. Biases are a short sorted
// list a row; each CTA looks through the part that can fall into its tokens
// (256 probes narrow a long list) and the thread at the first of a run of
// equal ids adds the run up into shared memory, so no order of atomics enters.
#include "kv_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 8 * kThreads;

struct RulesParams {
  const void* logits;
  size_t stride;
  int vocab;
  const uint32_t* seen;
  const uint16_t* counts;
  const float* rep;
  const float* freq;
  const float* pres;
  const int32_t* bias_start;
  const uint32_t* bias_ids;
  const float* bias_vals;
  int n_bias;
  const uint32_t* allowed;
  const int32_t* allowed_row;
  int n_allowed;
  void* out;
  size_t out_stride;
  unsigned long long* keys;
};

// F32: logits and output are float, else bf16. VEC: every row of every array
// starts on 16 bytes, so a full group of 8 is loaded whole.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kThreads) logits_rules_kernel(const RulesParams P) {
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  __shared__ __align__(16) float bias_s[kTokens];
  __shared__ unsigned long long key_s[kThreads / 32];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int i0 = blockIdx.x * kTokens + tid * 8;
  const int n = min(8, P.vocab - i0);  // tokens of this thread (may be <= 0)
  const size_t words = ((size_t)P.vocab + 31) / 32;
  const bool full = VEC && n == 8;

  float v[8];
  uint32_t seen = 0, allowed = 0xff;
  bool counted = false;
  uint16_t cnt[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  {
    const uint16_t* x16 = static_cast<const uint16_t*>(P.logits) + (size_t)b * P.stride + i0;
    const float* x32 = static_cast<const float*>(P.logits) + (size_t)b * P.stride + i0;
    if (full && F32) {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float4 u = reinterpret_cast<const float4*>(x32)[z];
        v[4 * z] = u.x;
        v[4 * z + 1] = u.y;
        v[4 * z + 2] = u.z;
        v[4 * z + 3] = u.w;
      }
    } else if (full) {
      const uint4 u = *reinterpret_cast<const uint4*>(x16);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = mc_bf16_to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] = i < n ? (F32 ? x32[i] : mc_bf16_to_f32(x16[i])) : -INFINITY;
    }
    if (P.counts) {
      const uint16_t* c = P.counts + (size_t)b * P.vocab + i0;
      if (full) {
        const uint4 u = *reinterpret_cast<const uint4*>(c);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) cnt[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        counted = (u.x | u.y | u.z | u.w) != 0;
      } else {
        counted = true;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) cnt[i] = c[i];
      }
    }
    if (n > 0) {
      if (P.seen) seen = reinterpret_cast<const uint8_t*>(P.seen + (size_t)b * words)[i0 / 8];
      if (P.allowed) {
        const int row = P.allowed_row ? P.allowed_row[b] : b;
        if (row >= 0 && row < P.n_allowed)
          allowed = reinterpret_cast<const uint8_t*>(P.allowed + (size_t)row * words)[i0 / 8];
      }
    }
  }

  const float rep = P.rep ? P.rep[b] : 1.0f;
  const float freq = P.freq ? P.freq[b] : 0.0f, pres = P.pres ? P.pres[b] : 0.0f;

  // ---- biases of this CTA's tokens
  bool biased = false;
  if (P.bias_start) {
    const int start = min(max(P.bias_start[b], 0), P.n_bias);
    const int end = min(max(P.bias_start[b + 1], start), P.n_bias);
    const uint32_t first = blockIdx.x * kTokens, last = first + kTokens;
    if (end > start) {
      biased = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) bias_s[tid + i * kThreads] = 0.0f;
      int lo = start, hi = end;
      if (end - start > 4 * kThreads) {
        // probes at every `step`-th entry bound the part with ids in [first, last)
        const int step = (end - start + kThreads - 1) / kThreads;
        const int at = start + tid * step;
        const uint32_t id = at < end ? P.bias_ids[at] : 0xffffffffu;
        const int below = __syncthreads_count(at < end && id < first);
        const int before = __syncthreads_count(at < end && id < last);
        lo = start + max(below - 1, 0) * step;
        hi = min(end, start + before * step);
      }
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kThreads) {
        const uint32_t id = P.bias_ids[j];
        const uint32_t back = P.bias_ids[max(j - 1, start)], next = P.bias_ids[min(j + 1, end - 1)];
        float sum = P.bias_vals[j];
        if (id < first || id >= last || (j > start && back == id)) continue;
        if (j + 1 < end && next == id)
          for (int e = j + 1; e < end && P.bias_ids[e] == id; ++e)
            sum = __fadd_rn(sum, P.bias_vals[e]);
        bias_s[id - first] = sum;
      }
      __syncthreads();
    }
  }

  if (seen) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (seen >> i & 1) v[i] = v[i] > 0.0f ? __fdiv_rn(v[i], rep) : __fmul_rn(v[i], rep);
  }
  if (counted) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (cnt[i]) v[i] = __fadd_rn(__fadd_rn(v[i], -__fmul_rn(freq, (float)cnt[i])), -pres);
  }
  if (biased) {
    const float4 u = reinterpret_cast<const float4*>(bias_s)[2 * tid];
    const float4 x = reinterpret_cast<const float4*>(bias_s)[2 * tid + 1];
    const float add[8] = {u.x, u.y, u.z, u.w, x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], add[i]);
  }
  if (allowed != 0xff) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(allowed >> i & 1)) v[i] = -INFINITY;
  }
  uint32_t packed[4];
  if (!F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(packed[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
      v[2 * i] = __uint_as_float(packed[i] << 16);
      v[2 * i + 1] = __uint_as_float(packed[i] & 0xffff0000u);
    }
  }
  uint16_t* o16 = static_cast<uint16_t*>(P.out) + (size_t)b * P.out_stride + i0;
  float* o32 = static_cast<float*>(P.out) + (size_t)b * P.out_stride + i0;
  if (full && F32) {
    reinterpret_cast<float4*>(o32)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(o32)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if (full) {
    *reinterpret_cast<uint4*>(o16) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= n) continue;
      if (F32) o32[i] = v[i];
      else o16[i] = (uint16_t)(__float_as_uint(v[i]) >> 16);
    }
  }
  if (!P.keys) return;
  // ---- the greedy key: the thread's largest value, the warp's, and the lowest index that has it
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, i < n ? v[i] : -INFINITY);  // NaN never wins
  bool any = top != -INFINITY;
  if (!any) {  // nothing, NaN, or -inf, which is a value too
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= i < n && v[i] == v[i];
  }
  const uint32_t mine = any ? mc_fkey(top) : 0u;
  const uint32_t most = __reduce_max_sync(0xffffffffu, mine);
  uint32_t at = 0xffffffffu;
  if (any && mine == most) {
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (i < n && v[i] == top) at = (uint32_t)(i0 + i);
  }
  at = __reduce_min_sync(0xffffffffu, at);
  if ((tid & 31) == 0) key_s[tid >> 5] = most ? (unsigned long long)most << 32 | (uint32_t)~at : 0;
  __syncthreads();
  if (tid == 0) {
    unsigned long long best = key_s[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) best = key_s[w] > best ? key_s[w] : best;
    if (best) atomicMax(P.keys + b, best);
  }
}

// One thread a row: rows are few, and two rows never share a word.
__global__ void __launch_bounds__(kThreads)
logits_mark_kernel(const uint32_t* __restrict__ tokens, int batch, uint32_t* seen,
                   uint16_t* counts, int vocab) {
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  const int b = blockIdx.x * kThreads + threadIdx.x;
  if (b >= batch) return;
  const uint32_t t = tokens[b];
  if (t >= (uint32_t)vocab) return;
  if (seen) seen[(size_t)b * (((size_t)vocab + 31) / 32) + t / 32] |= 1u << (t % 32);
  if (counts) {
    uint16_t* c = counts + (size_t)b * vocab + t;
    if (*c != 0xffff) *c += 1;
  }
}

}  // namespace

extern "C" int mc_logits_process(mc_ctx* ctx, const void* logits, size_t logits_stride, int dtype,
                                 int vocab, int batch, const uint32_t* seen,
                                 const uint16_t* counts, const float* repetition,
                                 const float* frequency, const float* presence,
                                 const int32_t* bias_start, const uint32_t* bias_ids,
                                 const float* bias_vals, int n_bias, const uint32_t* allowed,
                                 const int32_t* allowed_row, int n_allowed, void* out,
                                 size_t out_stride, unsigned long long* keys) {
  const char* name = "logits_process";
  MC_REQUIRE(dtype == MC_DTYPE_BF16 || dtype == MC_DTYPE_F32, "%s: logits dtype %d", name, dtype);
  MC_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "%s: vocab %d out of range", name, vocab);
  MC_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch %d out of range", name, batch);
  if (batch == 0) return MC_OK;
  MC_REQUIRE(logits && out, "%s: null pointer", name);
  MC_REQUIRE((repetition != nullptr) == (seen != nullptr),
             "%s: seen and repetition go together", name);
  MC_REQUIRE((counts != nullptr) == (frequency || presence),
             "%s: counts go with a frequency or presence penalty", name);
  // an empty list may come without addresses
  MC_REQUIRE(n_bias >= 0 && n_bias <= (1 << 30) &&
                 (bias_start ? n_bias == 0 || (bias_ids && bias_vals) : !bias_ids && !bias_vals),
             "%s: bias_start, bias_ids and bias_vals go together", name);
  MC_REQUIRE(!allowed || n_allowed >= 1, "%s: %d mask rows", name, n_allowed);
  MC_REQUIRE(allowed || !allowed_row, "%s: allowed_row without a mask", name);
  MC_REQUIRE(!allowed || allowed_row || n_allowed >= batch,
             "%s: %d mask rows for a batch of %d (allowed_row is null)", name, n_allowed, batch);
  const size_t size = dtype == MC_DTYPE_F32 ? 4 : 2, far = (size_t)1 << 40;
  MC_REQUIRE(mc_aligned(logits, size) && mc_aligned(out, size) && mc_aligned(keys, 8),
             "%s: misaligned rows or keys", name);
  MC_REQUIRE(logits_stride <= far && out_stride <= far, "%s: row stride out of range", name);
  MC_REQUIRE(batch <= 1 || out_stride >= (size_t)vocab, "%s: out rows overlap", name);
  const uintptr_t a = (uintptr_t)logits, c = (uintptr_t)out;
  const size_t a_bytes = size * ((size_t)(batch - 1) * logits_stride + vocab);
  const size_t c_bytes = size * ((size_t)(batch - 1) * out_stride + vocab);
  MC_REQUIRE((a == c && (logits_stride == out_stride || batch == 1)) || a + a_bytes <= c ||
                 c + c_bytes <= a,
             "%s: out overlaps logits without being logits", name);
  MC_REQUIRE(ctx, "%s: null context", name);
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  const RulesParams P{logits, logits_stride, vocab, seen, counts, repetition, frequency, presence,
                      bias_start, bias_ids, bias_vals, n_bias, allowed, allowed_row, n_allowed,
                      out, out_stride, keys};
  const bool rows16 = batch == 1 || (logits_stride * size % 16 == 0 && out_stride * size % 16 == 0);
  const bool vec = mc_aligned(logits, 16) && mc_aligned(out, 16) && rows16 &&
                   (!counts || (mc_aligned(counts, 16) && (batch == 1 || vocab % 8 == 0)));
  const dim3 grid((unsigned)(((size_t)vocab + kTokens - 1) / kTokens), (unsigned)batch);
  auto fn = dtype == MC_DTYPE_F32
                ? (vec ? logits_rules_kernel<true, true> : logits_rules_kernel<true, false>)
                : (vec ? logits_rules_kernel<false, true> : logits_rules_kernel<false, false>);
  MC_CUDA(mc_launch_pdl(fn, grid, dim3(kThreads), 0, ctx->stream, P));
  return mc_after_launch("logits_rules_kernel");
}

extern "C" int mc_logits_mark(mc_ctx* ctx, const uint32_t* tokens, int batch, uint32_t* seen,
                              uint16_t* counts, int vocab) {
  MC_REQUIRE(batch >= 0, "logits_mark: batch %d", batch);
  MC_REQUIRE(vocab >= 1, "logits_mark: vocab %d", vocab);
  if (batch == 0) return MC_OK;
  MC_REQUIRE(tokens && (seen || counts), "logits_mark: null pointer");
  MC_REQUIRE(ctx, "logits_mark: null context");
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  MC_CUDA(mc_launch_pdl(logits_mark_kernel, dim3((batch + kThreads - 1) / kThreads),
                        dim3(kThreads), 0, ctx->stream, tokens, batch, seen, counts, vocab));
  return mc_after_launch("logits_mark_kernel");
}
