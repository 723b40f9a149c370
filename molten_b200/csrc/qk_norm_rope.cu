// Norm and rotation of queries and keys, and the cache write, in one pass
// over a step's Q, K and V rows (mc_qk_norm_rope).
//
// For each head row x of a token at position p:
//   y = x / sqrt(mean(x^2) + eps) * w                    (w: per-dimension gain)
//   (a, b) -> (a cos - b sin, b cos + a sin), angle p * f_i, for the rot_dim/2
//   pairs (i, i + rot_dim/2) or, interleaved, (2i, 2i + 1)
// all in fp32, rounded once where it is stored: Q and a bf16 cache to bf16,
// an e4m3 cache to e4m3 of value / scale (saturating at +-448).
//
// The angle. p * f_i in fp32 is off by p * 2^-24 radians, 0.008 at position
// 131072: more than a bf16 step of the result. Each frequency is therefore
// given as a fraction of a turn in 64-bit fixed point, and p times it modulo
// 2^64 is the exact angle modulo a turn: one 64-bit multiply, whatever the
// position, and sincospi of the signed remainder.
//
// What bounds it: latency (the launch, the angles and first rows of a CTA, which
// nothing overlaps) and instructions, 52% of issue slots for a prompt's rows;
// each row is read once and written once. A thread holds 8 elements of one head
// row, the two groups of 4 that rotate into each other (so no pair crosses
// threads), for every token of the CTA's batch: its gains, addresses and role
// stay in registers. A batch's cosines, sines and cache rows are computed once
// into shared memory by all threads together. One wave of CTAs shares the
// tokens evenly, in batches of up to 16, with 4 tokens' loads in flight, each
// asked for as soon as the one in its place is unpacked (4096 tokens of 32 + 2
// x 8 heads of 64, 50 MB, of which the 25 MB that are read come from DRAM at a
// quarter of its rate: 12.7 us; 4 loaded together after 4 are done, in batches of 8, 14.6; 3 CTAs an SM
// with 2 in flight each 13.0; a CTA a token, rotation partners by shuffle,
// 25.6).
#include <cuda_fp8.h>
#include <math.h>

#include "kv_common.cuh"

namespace {

constexpr int kMaxThreads = 384;
constexpr int kBatch = 16;   // most tokens of a CTA
constexpr int kFlight = 4;    // tokens whose loads are in flight together
constexpr int kResident = 2;  // CTAs an SM holds at once

struct RopeParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;  // null: V is not written
  size_t q_stride, k_stride, v_stride;
  int tokens, share, batch;  // tokens of a CTA, and of them at once (1 to kBatch)
  int H, K, rows, group;  // rows = H + K (+ K with v), `group` of them a CTA
  const uint16_t* qw;  // null: no norm
  const uint16_t* kw;
  float eps;
  const int32_t* positions;
  const unsigned long long* turns;
  int rot, interleaved;
  uint16_t* q_out;
  size_t q_out_stride;
  const unsigned long long* slots;  // null: token t goes to slot t
  void* kc;
  void* vc;
  uint32_t n_slots, page_rows, block_size;
  const float* k_scale;
  const float* v_scale;
  uint32_t* status;
};

// Two floats under one instruction, each rounded as alone.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 parts(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// 4 elements: the even two and the odd two.
struct Four {
  Two even, odd;
};

__device__ __forceinline__ Four unpack4(const uint2& u) {
  return {two(__uint_as_float(u.x << 16), __uint_as_float(u.y << 16)),
          two(__uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y & 0xffff0000u))};
}

__device__ __forceinline__ uint2 pack4(const Four& f) {
  const float2 e = parts(f.even), o = parts(f.odd);
  uint2 r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.x) : "f"(o.x), "f"(e.x));
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.y) : "f"(o.y), "f"(e.y));
  return r;
}

__device__ __forceinline__ uint32_t pack4_e4m3(const Four& f) {
  const float2 e = parts(f.even), o = parts(f.odd);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(e.x, o.x), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(e.y, o.y), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// (a, b) -> (a cos - b sin, b cos + a sin); `minus`: -sin
__device__ __forceinline__ void rotate(Two& a, Two& b, Two cosine, Two sine, Two minus) {
  const Two p = a;
  a = fma2(b, minus, mul(p, cosine));
  b = fma2(p, sine, mul(b, cosine));
}

// D: head_dim; F8: e4m3 cache.
template <int D, bool F8>
__global__ void __launch_bounds__(kMaxThreads, kResident) qk_norm_rope_kernel(const RopeParams P) {
  constexpr int L = D / 8;  // threads of a row
  // cosines and sines of a token, those of a thread's 4 pairs together
  __shared__ __align__(16) float cos_s[kBatch][D / 2], sin_s[kBatch][D / 2];
  __shared__ uint32_t row_s[kBatch];  // the token's row of head 0 in the cache, all ones: none
  const int tid = threadIdx.x, c = tid % L;
  const int half = P.rot / 2, turned = P.rot / 8;  // threads of a row that rotate
  const int t_end = min(P.tokens, (int)(blockIdx.x + 1) * P.share);
  int t0 = blockIdx.x * P.share;

  // ---- this thread's row and its two groups of 4 elements
  const int r = blockIdx.y * P.group + tid / L;
  const bool in = r < P.rows && tid / L < P.group;
  const bool is_q = r < P.H, is_k = !is_q && r < P.H + P.K;
  const int h = is_q ? r : is_k ? r - P.H : r - P.H - P.K;
  const bool turns_here = (is_q || is_k) && c < turned;
  int a = 2 * c, b = 2 * c + 1;  // groups
  if (!P.interleaved && c < turned) {
    a = c;
    b = c + turned;
  }
  const uint16_t* src = is_q ? P.q : is_k ? P.k : P.v;
  const size_t stride = is_q ? P.q_stride : is_k ? P.k_stride : P.v_stride;
  src += (size_t)h * D;
  const uint16_t* w = is_q ? P.qw : is_k ? P.kw : nullptr;
  uint16_t* q_to = P.q_out + (size_t)t0 * P.q_out_stride + (size_t)h * D;
  void* cache = is_k ? P.kc : P.vc;
  const uint32_t head_row = (uint32_t)h * P.block_size;
  mc_pdl_launch_dependents();
  mc_pdl_wait();

  uint2 xa[kFlight], xb[kFlight];
  int coming = in ? t_end - t0 : 0;  // tokens that are still to be asked for, the next at src
  src += (size_t)t0 * stride;
  auto load = [&](int i) {
    if (coming > 0) {
      // plain loads: q_out may be q
      xa[i] = *reinterpret_cast<const uint2*>(src + 4 * a);
      xb[i] = *reinterpret_cast<const uint2*>(src + 4 * b);
    }
    --coming;
    src += stride;
  };
#pragma unroll
  for (int i = 0; i < kFlight; ++i) load(i);
  Four ga, gb;
  if (in && w) {
    ga = unpack4(__ldg(reinterpret_cast<const uint2*>(w) + a));
    gb = unpack4(__ldg(reinterpret_cast<const uint2*>(w) + b));
  }
  float scale = 1.0f;
  if (F8 && in && !is_q) {
    const float* s = is_k ? P.k_scale : P.v_scale;
    if (s) scale = __fdiv_rn(1.0f, s[h]);
  }
  for (; t0 < t_end; t0 += P.batch) {
    const int n = min(P.batch, t_end - t0);
    __syncthreads();  // the batch before is done with the shared arrays
    for (int i = tid; i < n * half; i += blockDim.x) {
      const int t = i / half, f = i - t * half;
      const unsigned long long turn =
          (unsigned long long)(long long)P.positions[t0 + t] * P.turns[f];
      // signed fraction of a turn in [-1/2, 1/2), doubled: half turns
      const float x = __ll2float_rn((long long)turn) * 1.0842021724855044e-19f;  // 2^-63
      float s, co;
      sincospif(x, &s, &co);
      // a thread's pairs 0 1 2 3 stand as two words of two that rotate under one instruction:
      // 0 2 and 1 3, interleaved 0 1 and 2 3
      const int at = P.interleaved || f % 4 == 0 || f % 4 == 3 ? f : f ^ 3;
      cos_s[t][at] = co;
      sin_s[t][at] = s;
    }
    if (tid < n) {
      const unsigned long long slot = P.slots ? P.slots[t0 + tid] : (unsigned long long)(t0 + tid);
      uint32_t row = 0xffffffffu;
      if (slot < P.n_slots) {
        const uint32_t page = (uint32_t)slot / P.block_size;
        row = page * P.page_rows + ((uint32_t)slot - page * P.block_size);
      } else if (slot != MC_KV_SLOT_NONE && P.status && blockIdx.y == 0) {
        atomicOr(P.status, MC_KV_BAD_SLOT);
      }
      row_s[tid] = row;
    }
    __syncthreads();

    for (int t = 0; t < n; t += kFlight) {
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        if (t + i >= n) break;  // the same for the whole CTA
        Four x = unpack4(xa[i]), y = unpack4(xb[i]);
        load(i);
        if (P.qw || P.kw) {
          const float2 sum = parts(fma2(
              x.even, x.even,
              fma2(x.odd, x.odd, fma2(y.even, y.even, mul(y.odd, y.odd)))));
          float ss = sum.x + sum.y;
#pragma unroll
          for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
          if (w) {
            const float one = rsqrtf(__fmaf_rn(ss, 1.0f / D, P.eps));
            const Two inv = two(one, one);
            x = {mul(mul(x.even, inv), ga.even), mul(mul(x.odd, inv), ga.odd)};
            y = {mul(mul(y.even, inv), gb.even), mul(mul(y.odd, inv), gb.odd)};
          }
        }
        if (turns_here) {
          // this thread's four frequencies: 4 c .. 4 c + 3
          const float4 e = *reinterpret_cast<const float4*>(&cos_s[t + i][4 * c]);
          const float4 f = *reinterpret_cast<const float4*>(&sin_s[t + i][4 * c]);
          const Two c0 = two(e.x, e.y), c1 = two(e.z, e.w), s0 = two(f.x, f.y), s1 = two(f.z, f.w);
          const Two m0 = two(-f.x, -f.y), m1 = two(-f.z, -f.w);
          if (P.interleaved) {
            rotate(x.even, x.odd, c0, s0, m0);
            rotate(y.even, y.odd, c1, s1, m1);
          } else {
            rotate(x.even, y.even, c0, s0, m0);
            rotate(x.odd, y.odd, c1, s1, m1);
          }
        }
        if (!in) continue;
        if (is_q) {
          *reinterpret_cast<uint2*>(q_to + 4 * a) = pack4(x);
          *reinterpret_cast<uint2*>(q_to + 4 * b) = pack4(y);
          q_to += P.q_out_stride;
        } else if (row_s[t + i] != 0xffffffffu) {
          const size_t at = (size_t)(row_s[t + i] + head_row) * D;
          if (F8) {
            const Two by = two(scale, scale);
            x = {mul(x.even, by), mul(x.odd, by)};
            y = {mul(y.even, by), mul(y.odd, by)};
            uint8_t* to = static_cast<uint8_t*>(cache) + at;
            *reinterpret_cast<uint32_t*>(to + 4 * a) = pack4_e4m3(x);
            *reinterpret_cast<uint32_t*>(to + 4 * b) = pack4_e4m3(y);
          } else {
            uint16_t* to = static_cast<uint16_t*>(cache) + at;
            *reinterpret_cast<uint2*>(to + 4 * a) = pack4(x);
            *reinterpret_cast<uint2*>(to + 4 * b) = pack4(y);
          }
        }
      }
    }
  }
}

template <int D, bool F8>
int launch_rope(mc_ctx* ctx, RopeParams& P) {
  // rows of a token: even parts of at most kMaxThreads threads
  const int most = kMaxThreads / (D / 8), parts = (P.rows + most - 1) / most;
  P.group = (P.rows + parts - 1) / parts;
  const int threads = (P.group * (D / 8) + 31) / 32 * 32;
  // one wave: equal shares of the tokens for every CTA that fits (at least one, where the parts
  // alone are more than a wave), in equal batches
  const int wave = kResident * ctx->num_sms, slots = wave > parts ? wave / parts : 1;
  P.share = (P.tokens + slots - 1) / slots;
  const int batches = (P.share + kBatch - 1) / kBatch;
  // whole rounds of the tokens in flight, so that a token keeps its place among them
  P.batch = ((P.share + batches - 1) / batches + kFlight - 1) / kFlight * kFlight;
  const dim3 grid((unsigned)((P.tokens + P.share - 1) / P.share), (unsigned)parts);
  MC_CUDA(mc_launch_pdl(qk_norm_rope_kernel<D, F8>, grid, dim3(threads), 0, ctx->stream, P));
  return mc_after_launch("qk_norm_rope_kernel");
}

// [p, p + bytes) and [q, q + more) share a byte
bool overlap(const void* p, size_t bytes, const void* q, size_t more) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + more && b < a + bytes;
}

// Of `tokens` rows (or pages) of `an` bytes at a and of `bn` bytes at b, one each `a_step` / `b_step` bytes,
// some share a byte. Rows of one step may interleave (parts of one fused row); of two steps,
// their whole ranges count.
bool rows_overlap(const void* a, size_t an, size_t a_step, const void* b, size_t bn, size_t b_step,
                  size_t tokens) {
  if (!overlap(a, (tokens - 1) * a_step + an, b, (tokens - 1) * b_step + bn)) return false;
  if (tokens == 1 || a_step != b_step || a_step == 0) return true;
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  const size_t behind = y >= x ? (y - x) % a_step : (a_step - (x - y) % a_step) % a_step;
  return behind < an || behind + bn > a_step;
}

}  // namespace

extern "C" int mc_rope_turns(float theta, float position_scale, int rot_dim, uint64_t* out) {
  MC_REQUIRE(rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= 1024, "rope_turns: rot_dim %d",
             rot_dim);
  MC_REQUIRE(isfinite(theta) && theta > 0.0f, "rope_turns: theta must be positive");
  MC_REQUIRE(isfinite(position_scale) && position_scale >= 0.0f,
             "rope_turns: position_scale must not be negative");
  MC_REQUIRE(out, "rope_turns: null out");
  for (int i = 0; i < rot_dim / 2; ++i) {
    const double f = (double)position_scale * pow((double)theta, -2.0 * i / rot_dim);
    const double turns = f / 6.283185307179586476925286766559;
    // the fraction of a turn times 2^64 (rounding up to a whole turn wraps to 0)
    const double fixed = rint((turns - floor(turns)) * 18446744073709551616.0);
    out[i] = fixed >= 18446744073709551616.0 ? 0 : (uint64_t)fixed;
  }
  return MC_OK;
}

extern "C" int mc_qk_norm_rope(mc_ctx* ctx, const uint16_t* q, size_t q_stride, const uint16_t* k,
                               size_t k_stride, const uint16_t* v, size_t v_stride, int n_tokens,
                               int n_heads, int n_kv_heads, int head_dim,
                               const uint16_t* q_norm_w, const uint16_t* k_norm_w, float eps,
                               const int32_t* positions, const uint64_t* turns, int rot_dim,
                               int interleaved, uint16_t* q_out, size_t q_out_stride,
                               const uint64_t* slots, void* k_cache, void* v_cache, int kv_dtype,
                               int num_blocks, int block_size, size_t block_stride,
                               const float* k_scale, const float* v_scale, uint32_t* status) {
  const char* name = "qk_norm_rope";
  int rc = mc_check_kv_cache(name, k_cache, v_cache, kv_dtype, num_blocks, block_size,
                             block_stride, n_kv_heads, head_dim, k_scale, v_scale);
  if (rc) return rc;
  MC_REQUIRE(n_tokens >= 0 && n_tokens <= (1 << 30), "%s: n_tokens %d out of range", name, n_tokens);
  if (n_tokens == 0) return MC_OK;
  MC_REQUIRE(n_heads >= 1 && n_heads <= 16384, "%s: n_heads %d out of range", name, n_heads);
  MC_REQUIRE(rot_dim >= 0 && rot_dim % 16 == 0 && rot_dim <= head_dim,
             "%s: rot_dim %d must be a multiple of 16 up to head_dim", name, rot_dim);
  MC_REQUIRE(isfinite(eps) && eps >= 0.0f, "%s: eps must be finite and not negative", name);
  MC_REQUIRE(q && k && q_out && (rot_dim == 0 || (positions && turns)), "%s: null pointer", name);
  MC_REQUIRE(mc_aligned(q, 16) && mc_aligned(k, 16) && mc_aligned(v, 16) && mc_aligned(q_out, 16) &&
                 mc_aligned(q_norm_w, 16) && mc_aligned(k_norm_w, 16),
             "%s: rows and gains must be 16-byte aligned", name);
  MC_REQUIRE(mc_aligned(turns, 8) && mc_aligned(slots, 8), "%s: turns/slots misaligned", name);
  const size_t qn = (size_t)n_heads * head_dim, kn = (size_t)n_kv_heads * head_dim;
  MC_REQUIRE(q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && q_out_stride % 8 == 0,
             "%s: token strides must be multiples of 8 elements", name);
  const size_t far = (size_t)1 << 40;
  MC_REQUIRE(q_stride <= far && k_stride <= far && v_stride <= far && q_out_stride <= far,
             "%s: token stride out of range", name);
  MC_REQUIRE(n_tokens <= 1 || q_out_stride >= qn, "%s: q_out rows overlap", name);
  const size_t T = (size_t)n_tokens, q_step = 2 * q_stride, out_step = 2 * q_out_stride;
  // q_out may be q itself (a lane writes the 16 bytes it read), nothing else that is read
  MC_REQUIRE((q_out == q && (q_out_stride == q_stride || T == 1)) ||
                 !rows_overlap(q_out, 2 * qn, out_step, q, 2 * qn, q_step, T),
             "%s: q_out overlaps q without being q", name);
  MC_REQUIRE(!rows_overlap(q_out, 2 * qn, out_step, k, 2 * kn, 2 * k_stride, T) &&
                 !rows_overlap(q_out, 2 * qn, out_step, v, 2 * kn, 2 * v_stride, T),
             "%s: q_out overlaps k or v", name);
  const size_t size = kv_dtype == MC_DTYPE_BF16 ? 2 : 1;  // bytes of an element
  const size_t cache_bytes = size * (block_stride * ((size_t)num_blocks - 1) +
                                     (size_t)n_kv_heads * block_size * head_dim);
  // K's and V's pages may alternate, but share no byte (V NULL: one may stand for both)
  const size_t page_bytes = size * ((size_t)n_kv_heads * block_size * head_dim);
  MC_REQUIRE(!v || !rows_overlap(k_cache, page_bytes, size * block_stride, v_cache, page_bytes,
                                 size * block_stride, (size_t)num_blocks),
             "%s: k_cache overlaps v_cache", name);
  const void* const rows[4] = {q, k, v, q_out};
  const size_t bytes[4] = {2 * qn, 2 * kn, 2 * kn, 2 * qn};
  const size_t steps[4] = {q_step, 2 * k_stride, 2 * v_stride, out_step};
  for (int i = 0; i < 4; ++i) {
    const size_t n = (T - 1) * steps[i] + bytes[i];
    MC_REQUIRE(!overlap(rows[i], n, k_cache, cache_bytes) &&
                   !overlap(rows[i], n, v_cache, cache_bytes),
               "%s: q, k, v or q_out lies in the cache", name);
  }
  MC_REQUIRE(ctx, "%s: null context", name);
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  RopeParams P{q, k, v, q_stride, k_stride, v_stride, n_tokens, 1, 1, n_heads, n_kv_heads,
               n_heads + n_kv_heads * (v ? 2 : 1), 0, q_norm_w, k_norm_w, eps, positions,
               reinterpret_cast<const unsigned long long*>(turns), rot_dim, interleaved, q_out,
               q_out_stride, reinterpret_cast<const unsigned long long*>(slots), k_cache, v_cache,
               (uint32_t)num_blocks * (uint32_t)block_size, (uint32_t)(block_stride / head_dim),
               (uint32_t)block_size, k_scale, v_scale, status};
  const bool f8 = kv_dtype == MC_DTYPE_E4M3;
  if (head_dim == 64) return f8 ? launch_rope<64, true>(ctx, P) : launch_rope<64, false>(ctx, P);
  return f8 ? launch_rope<128, true>(ctx, P) : launch_rope<128, false>(ctx, P);
}
