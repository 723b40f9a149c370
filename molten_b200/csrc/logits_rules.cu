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
// What bounds it: bytes (2 to 8 read and 2 or 4 written a token) and, with
// every rule on, instructions, some 40 a token and lane. A thread takes 8
// tokens: one 16-byte load of bf16 logits, one of counts, one byte of each
// bitmap, the next span's on their way while it works on one (48 rows of
// 128000, 38 MB with all rules, of which the 26 MB that are read come from
// DRAM: 13.6 us; without biases and penalties, 25 MB, 8.0 us; two spans ahead
// 1 us more). A CTA takes a few spans of 2048 tokens of one row, so that a
// large batch is one wave. Biases are a short
// sorted list a row; each CTA looks through the part that can fall into its
// tokens (256 probes narrow a long list) and the thread at the first of a run
// of equal ids adds the run up into shared memory, so no order of atomics
// enters; the list is on its way while that memory is zeroed (0.5 us).
#include "kv_common.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kSpan = 8 * kThreads;  // tokens a CTA takes at once
constexpr int kSpans = 4;            // most spans of a CTA
constexpr int kSpansBiased = 5;      // with biases, in one wave
constexpr int kResident = 5;         // CTAs an SM holds at once

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
  int spans;
};

// The 8 logits of one thread's group, as stored, with what the rules say about them.
template <bool F32>
struct Group {
  uint32_t x[F32 ? 8 : 4];
  uint32_t cnt[4];         // counts, two a word
  uint32_t seen, allowed;  // a bit each
};

// Bits i .. i + 7 of a bitmap of `bytes` bytes (i from -7 on; bits outside are 0).
__device__ __forceinline__ uint32_t bits8(const uint8_t* map, int i, int bytes) {
  const int at = i >> 3, sh = i & 7;
  uint32_t w = i >= 0 ? map[at] : 0u;
  if (sh && at + 1 < bytes) w |= (uint32_t)map[at + 1] << 8;
  return w >> sh & 0xffu;
}

// F32: logits and output are float, else bf16. VEC: the rows of logits, output
// and counts all start equally far behind a 16-byte border (`shift` elements,
// another number for each row of an odd vocabulary): groups of 8 begin at the
// borders, and all but a row's first and last are loaded whole.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kThreads, kResident) logits_rules_kernel(const RulesParams P) {
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  extern __shared__ __align__(16) float bias_s[];  // [spans * kSpan] where there are biases
  __shared__ unsigned long long key_s[kThreads / 32];
  const int b = blockIdx.y, tid = threadIdx.x;
  const size_t words = ((size_t)P.vocab + 31) / 32;
  const uint16_t* x16 = static_cast<const uint16_t*>(P.logits) + (size_t)b * P.stride;
  const float* x32 = static_cast<const float*>(P.logits) + (size_t)b * P.stride;
  uint16_t* o16 = static_cast<uint16_t*>(P.out) + (size_t)b * P.out_stride;
  float* o32 = static_cast<float*>(P.out) + (size_t)b * P.out_stride;
  const uint16_t* counts = P.counts + (size_t)b * P.vocab;
  const int shift = !VEC ? 0 : F32 ? (int)((uintptr_t)x32 / 4 % 4) : (int)((uintptr_t)x16 / 2 % 8);
  const int first = blockIdx.x * P.spans * kSpan - shift;  // of this CTA; may be below 0
  const uint8_t* seen =
      P.seen ? reinterpret_cast<const uint8_t*>(P.seen + (size_t)b * words) : nullptr;
  const uint8_t* allowed = nullptr;
  if (P.allowed) {
    const int row = P.allowed_row ? P.allowed_row[b] : b;
    if (row >= 0 && row < P.n_allowed)
      allowed = reinterpret_cast<const uint8_t*>(P.allowed + (size_t)row * words);
  }
  const float rep = P.rep ? P.rep[b] : 1.0f, inv = __fdiv_rn(1.0f, rep);  // as mc_sample_draw
  const float freq = P.freq ? P.freq[b] : 0.0f, pres = P.pres ? P.pres[b] : 0.0f;

  auto load = [&](Group<F32>& w, int z) {
    const int i1 = first + z * kSpan + tid * 8;
    w.seen = 0;
    w.allowed = 0xff;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.cnt[i] = 0;
    if (z >= P.spans || i1 >= P.vocab) return;
    if (VEC && i1 >= 0 && i1 + 8 <= P.vocab) {
#pragma unroll
      for (int i = 0; i < (F32 ? 2 : 1); ++i) {
        const uint4 u = F32 ? reinterpret_cast<const uint4*>(x32 + i1)[i]
                            : *reinterpret_cast<const uint4*>(x16 + i1);
        w.x[4 * i] = u.x;
        w.x[4 * i + 1] = u.y;
        w.x[4 * i + 2] = u.z;
        w.x[4 * i + 3] = u.w;
      }
      if (P.counts) {
        uint2 c[2];  // rows of float logits begin on 8 bytes of counts
        if (F32) {
          c[0] = *reinterpret_cast<const uint2*>(counts + i1);
          c[1] = *reinterpret_cast<const uint2*>(counts + i1 + 4);
        } else {
          const uint4 u = *reinterpret_cast<const uint4*>(counts + i1);
          c[0] = make_uint2(u.x, u.y);
          c[1] = make_uint2(u.z, u.w);
        }
        w.cnt[0] = c[0].x;
        w.cnt[1] = c[0].y;
        w.cnt[2] = c[1].x;
        w.cnt[3] = c[1].y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < (F32 ? 8 : 4); ++i) w.x[i] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i1 + i < 0 || i1 + i >= P.vocab) continue;
        if (F32) w.x[i] = __float_as_uint(x32[i1 + i]);
        else w.x[i / 2] |= (uint32_t)x16[i1 + i] << (16 * (i & 1));
        if (P.counts) w.cnt[i / 2] |= (uint32_t)counts[i1 + i] << (16 * (i & 1));
      }
    }
    if (shift == 0) {
      if (seen) w.seen = seen[i1 / 8];
      if (allowed) w.allowed = allowed[i1 / 8];
    } else {
      if (seen) w.seen = bits8(seen, i1, (int)(4 * words));
      if (allowed) w.allowed = bits8(allowed, i1, (int)(4 * words));
    }
  };

  Group<F32> w, next;
  load(w, 0);

  // ---- biases of this CTA's tokens
  bool biased = false;
  if (P.bias_start) {
    const int from = P.bias_start[b], to = P.bias_start[b + 1];
    for (int i = 0; i < 2 * P.spans; ++i)
      reinterpret_cast<float4*>(bias_s)[tid + i * kThreads] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int start = min(max(from, 0), P.n_bias), end = min(max(to, start), P.n_bias);
    const uint32_t low = (uint32_t)max(first, 0), last = (uint32_t)(first + P.spans * kSpan);
    if (end > start) {
      biased = true;
      int lo = start, hi = end;
      if (end - start > 4 * kThreads) {
        // probes at every `step`-th entry bound the part with ids in [low, last)
        const int step = (end - start + kThreads - 1) / kThreads;
        const int at = start + tid * step;
        const uint32_t id = at < end ? P.bias_ids[at] : 0xffffffffu;
        const int below = __syncthreads_count(at < end && id < low);
        const int before = __syncthreads_count(at < end && id < last);
        lo = start + max(below - 1, 0) * step;
        hi = min(end, start + before * step);
      }
      bool zeroed = false;  // by all threads
      for (int j0 = lo; j0 < hi; j0 += kThreads) {
        const int j = min(j0 + tid, hi - 1);
        const uint32_t id = P.bias_ids[j];
        const uint32_t back = P.bias_ids[max(j - 1, start)], ahead = P.bias_ids[min(j + 1, end - 1)];
        float sum = P.bias_vals[j];
        if (!zeroed) __syncthreads();
        zeroed = true;
        if (j0 + tid >= hi || id < low || id >= last || (j > start && back == id)) continue;
        if (j + 1 < end && ahead == id)
          for (int e = j + 1; e < end && P.bias_ids[e] == id; ++e)
            sum = __fadd_rn(sum, P.bias_vals[e]);
        bias_s[(int)id - first] = sum;
      }
      __syncthreads();
    }
  }

  float top = -INFINITY;  // this thread's largest value and the first group that has it (NaN
  int best_z = -1;        // never wins)
  auto apply = [&](const Group<F32>& w, int z) {
    const int i1 = first + z * kSpan + tid * 8;
    if (i1 >= P.vocab) return;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = __uint_as_float(F32     ? w.x[i]
                             : i & 1 ? w.x[i / 2] & 0xffff0000u
                                     : w.x[i / 2] << 16);
    if (w.seen) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float by = v[i] > 0.0f ? inv : rep;
        v[i] = __fmul_rn(v[i], w.seen >> i & 1 ? by : 1.0f);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t two = w.cnt[i / 2];
      if (two == 0) continue;
      const float c0 = (float)(two & 0xffffu), c1 = (float)(two >> 16);
      if (two & 0xffffu) v[i] = __fadd_rn(__fadd_rn(v[i], -__fmul_rn(freq, c0)), -pres);
      if (two >> 16) v[i + 1] = __fadd_rn(__fadd_rn(v[i + 1], -__fmul_rn(freq, c1)), -pres);
    }
    if (biased) {
      const float4* add = reinterpret_cast<const float4*>(bias_s + z * kSpan + tid * 8);
      const float4 u = add[0], x = add[1];
      const float f[8] = {u.x, u.y, u.z, u.w, x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], f[i]);
    }
    if (w.allowed != 0xff) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(w.allowed >> i & 1)) v[i] = -INFINITY;
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
    const bool full = i1 >= 0 && i1 + 8 <= P.vocab;
    if (VEC && full) {
      if (F32) {
        *reinterpret_cast<float4*>(o32 + i1) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(o32 + i1 + 4) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(o16 + i1) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i1 + i < 0 || i1 + i >= P.vocab) {
          v[i] = __uint_as_float(0x7fc00000u);  // never the largest
          continue;
        }
        if (F32) o32[i1 + i] = v[i];
        else o16[i1 + i] = (uint16_t)(__float_as_uint(v[i]) >> 16);
      }
    }
    if (P.keys) {
      const float most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])),
                               fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
      if (most > top || (best_z < 0 && most == most)) {
        top = most;
        best_z = z;
      }
    }
  };

  for (int z = 0; z < P.spans; ++z) {
    load(next, z + 1);  // on its way while this span is worked on
    apply(w, z);
    w = next;
  }
  if (!P.keys) return;
  // ---- the greedy key: the warp's largest value; who has it reads its group again for the
  // lowest token
  const uint32_t mine = best_z >= 0 ? mc_fkey(top) : 0u;
  const uint32_t most = __reduce_max_sync(0xffffffffu, mine);
  uint32_t at = 0xffffffffu;
  if (mine == most && most) {
    const int i1 = first + best_z * kSpan + tid * 8;
#pragma unroll
    for (int i = 7; i >= 0; --i)
      if (i1 + i >= 0 && i1 + i < P.vocab &&
          (F32 ? o32[i1 + i] : mc_bf16_to_f32(o16[i1 + i])) == top)
        at = (uint32_t)(i1 + i);
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
  MC_REQUIRE(mc_aligned(logits, size) && mc_aligned(out, size) && mc_aligned(keys, 8) &&
                 mc_aligned(counts, 2),
             "%s: misaligned rows, counts or keys", name);
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
  RulesParams P{logits, logits_stride, vocab, seen, counts, repetition, frequency, presence,
                bias_start, bias_ids, bias_vals, n_bias, allowed, allowed_row, n_allowed,
                out, out_stride, keys, 1};
  // every row's start the same number of elements behind a 16-byte border (counts: 8 bytes
  // for float logits, whose groups begin on those)
  const size_t lane = 16 / size, la = (uintptr_t)logits / size % lane;
  const bool vec = (uintptr_t)out / size % lane == la &&
                   (batch == 1 || logits_stride % lane == out_stride % lane) &&
                   (!counts || ((uintptr_t)counts / 2 % lane == la && mc_aligned(counts, 2) &&
                                (batch == 1 || (size_t)vocab % lane == logits_stride % lane)));
  // CTAs a row: as many as one wave leaves it, in runs of at most 4 spans; 5 with biases where that
  // makes one wave, since a second one would zero and fill its shared memory once more. With the
  // token tail, runs of 5 and of 4: one wave by fives, two by fours: 50 rows of 128000 16.4 and 17.6
  // us, 56 of 128000 16.0 and 18.3, 100 of 65536 16.7 and 18.5; two waves either way: 64 of 128000
  // 21.1 and 19.8, 128 of 65536 22.3 and 21.4, 256 of 32000 23.5 and 21.3; without biases 48 of
  // 128000 15.2 and 14.6, 128 of 128000 28.9 and 27.2 (by threes 30.2). 5 spans are the most whose
  // shared memory (8 KB each) kResident CTAs hold.
  const int all = (vocab + (vec ? (int)lane - 1 : 0) + kSpan - 1) / kSpan;
  const int share = kResident * ctx->num_sms / batch;
  const int spans_of_a_wave = share > 0 ? (all + share - 1) / share : all;
  const int spans = spans_of_a_wave <= (bias_start ? kSpansBiased : kSpans) ? spans_of_a_wave : kSpans;
  P.spans = spans;
  const dim3 grid((unsigned)((all + spans - 1) / spans), (unsigned)batch);
  auto fn = dtype == MC_DTYPE_F32
                ? (vec ? logits_rules_kernel<true, true> : logits_rules_kernel<true, false>)
                : (vec ? logits_rules_kernel<false, true> : logits_rules_kernel<false, false>);
  const size_t smem = bias_start ? (size_t)spans * kSpan * sizeof(float) : 0;
  MC_CUDA(mc_launch_pdl(fn, grid, dim3(kThreads), smem, ctx->stream, P));
  return mc_after_launch("logits_rules_kernel");
}

extern "C" int mc_logits_mark(mc_ctx* ctx, const uint32_t* tokens, int batch, uint32_t* seen,
                              uint16_t* counts, int vocab) {
  MC_REQUIRE(batch >= 0, "logits_mark: batch %d", batch);
  MC_REQUIRE(vocab >= 1, "logits_mark: vocab %d", vocab);
  if (batch == 0) return MC_OK;
  MC_REQUIRE(tokens && (seen || counts), "logits_mark: null pointer");
  MC_REQUIRE(mc_aligned(tokens, 4) && mc_aligned(seen, 4) && mc_aligned(counts, 2),
             "logits_mark: misaligned tokens, seen or counts");
  MC_REQUIRE(ctx, "logits_mark: null context");
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  MC_CUDA(mc_launch_pdl(logits_mark_kernel, dim3((batch + kThreads - 1) / kThreads),
                        dim3(kThreads), 0, ctx->stream, tokens, batch, seen, counts, vocab));
  return mc_after_launch("logits_mark_kernel");
}
