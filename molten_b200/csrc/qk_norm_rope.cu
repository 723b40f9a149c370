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
// What bounds it: bytes (each row read once, written once), and latency at a
// few tokens. A CTA takes one token: its threads first have the row loads in
// flight (16 bytes a lane, head_dim/8 lanes a row), then compute the token's
// cosines and sines once into shared memory for all its heads, then
// normalise (a shuffle reduction inside the row's lanes) and rotate (the
// partner 16 bytes come by shuffle).
#include <cuda_fp8.h>
#include <math.h>

#include "kv_common.cuh"

namespace {

constexpr int kMaxThreads = 512;

struct RopeParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;  // null: V is not written
  size_t q_stride, k_stride, v_stride;
  int H, K, rows;  // rows = H + K (+ K with v)
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
  int num_blocks, block_size;
  size_t block_stride;
  const float* k_scale;
  const float* v_scale;
  uint32_t* status;
};

__device__ __forceinline__ void unpack8(const uint4& u, float* f) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = mc_bf16_to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}

__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)mc_f32_to_bf16(f[2 * i]) | ((uint32_t)mc_f32_to_bf16(f[2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint2 pack8_e4m3(const float* f) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_fp8x2_storage_t b =
        __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    w[i >> 1] |= (uint32_t)b << (16 * (i & 1));
  }
  return make_uint2(w[0], w[1]);
}

// D: head_dim; F8: e4m3 cache.
template <int D, bool F8>
__global__ void __launch_bounds__(kMaxThreads) qk_norm_rope_kernel(const RopeParams P) {
  constexpr int L = D / 8;  // lanes of a row
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  __shared__ float2 cs[D / 2];
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31, c = lane % L;
  const int half = P.rot / 2, hc = P.rot / 16;  // 16-byte chunks of half the rotated part
  const int per_pass = blockDim.x / L;
  const unsigned long long slot = P.slots ? P.slots[t] : (unsigned long long)t;
  const unsigned long long n_slots = (unsigned long long)P.num_blocks * P.block_size;
  const bool store = slot < n_slots;
  if (!store && slot != MC_KV_SLOT_NONE && threadIdx.x == 0 && P.status)
    atomicOr(P.status, MC_KV_BAD_SLOT);
  const size_t page = store ? (size_t)(slot / P.block_size) * P.block_stride : 0;
  const int off = store ? (int)(slot % P.block_size) : 0;

  // every thread runs every pass: the shuffles need whole warps
  for (int r0 = 0; r0 < P.rows; r0 += per_pass) {
    const int r = r0 + threadIdx.x / L;
    const bool in = r < P.rows;
    const bool is_q = r < P.H, is_k = !is_q && r < P.H + P.K;
    const int h = is_q ? r : is_k ? r - P.H : r - P.H - P.K;
    uint4 raw = make_uint4(0, 0, 0, 0), wraw = make_uint4(0, 0, 0, 0);
    const uint16_t* w = is_q ? P.qw : is_k ? P.kw : nullptr;
    if (in) {
      const uint16_t* src = is_q   ? P.q + (size_t)t * P.q_stride
                            : is_k ? P.k + (size_t)t * P.k_stride
                                   : P.v + (size_t)t * P.v_stride;
      raw = reinterpret_cast<const uint4*>(src + (size_t)h * D)[c];  // q_out may be q
      if (w) wraw = __ldg(reinterpret_cast<const uint4*>(w) + c);
    }
    if (r0 == 0) {
      for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const unsigned long long turn =
            (unsigned long long)(long long)P.positions[t] * P.turns[i];
        // signed fraction of a turn in [-1/2, 1/2), doubled: half turns
        const float x = __ll2float_rn((long long)turn) * 1.0842021724855044e-19f;  // 2^-63
        float s, co;
        sincospif(x, &s, &co);
        cs[i] = make_float2(co, s);
      }
      __syncthreads();
    }
    float x[8];
    unpack8(raw, x);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(x[i], x[i], ss);
#pragma unroll
    for (int m = 1; m < L; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    if (w) {
      const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(ss, 1.0f / D, P.eps)));
      float g[8];
      unpack8(wraw, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * g[i];
    }
    // the other chunk of a half-split pair: c + hc or c - hc
    const int pc = c < hc ? c + hc : c < 2 * hc ? c - hc : c;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], (lane - c) + pc);
    if (is_q || is_k) {
      if (P.interleaved) {
        if (c < 2 * hc) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 e = cs[c * 4 + i];
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = __fmaf_rn(a, e.x, -(b * e.y));
            x[2 * i + 1] = __fmaf_rn(b, e.x, a * e.y);
          }
        }
      } else if (c < 2 * hc) {
        const bool first = c < hc;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 e = cs[(first ? c : c - hc) * 8 + i];
          x[i] = first ? __fmaf_rn(x[i], e.x, -(o[i] * e.y)) : __fmaf_rn(x[i], e.x, o[i] * e.y);
        }
      }
    }
    if (!in) continue;
    if (is_q) {
      reinterpret_cast<uint4*>(P.q_out + (size_t)t * P.q_out_stride + (size_t)h * D)[c] = pack8(x);
    } else if (store) {
      const size_t at = page + ((size_t)h * P.block_size + off) * D + 8 * c;
      void* cache = is_k ? P.kc : P.vc;
      if (F8) {
        const float* scale = is_k ? P.k_scale : P.v_scale;
        if (scale) {
          const float s = scale[h];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = __fdiv_rn(x[i], s);
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + at) = pack8_e4m3(x);
      } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + at) = pack8(x);
      }
    }
  }
}

template <int D, bool F8>
int launch_rope(mc_ctx* ctx, const RopeParams& P, int n_tokens) {
  int threads = ((P.rows * (D / 8) + 31) / 32) * 32;
  if (threads > kMaxThreads) threads = kMaxThreads;
  MC_CUDA(mc_launch_pdl(qk_norm_rope_kernel<D, F8>, dim3(n_tokens), dim3(threads), 0, ctx->stream,
                        P));
  return mc_after_launch("qk_norm_rope_kernel");
}

// [p, p + bytes) and [q, q + more) share a byte
bool overlap(const void* p, size_t bytes, const void* q, size_t more) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && a < b + more && b < a + bytes;
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
  MC_REQUIRE(n_tokens >= 0, "%s: n_tokens %d", name, n_tokens);
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
  const size_t T = (size_t)n_tokens - 1;
  const size_t q_bytes = 2 * (T * q_stride + qn), out_bytes = 2 * (T * q_out_stride + qn);
  // q_out may be q itself (a lane writes the 16 bytes it read), nothing else that is read
  MC_REQUIRE((q_out == q && (q_out_stride == q_stride || n_tokens == 1)) ||
                 !overlap(q_out, out_bytes, q, q_bytes),
             "%s: q_out overlaps q without being q", name);
  // parts of one fused row interleave: only a contiguous q_out can be judged against k and v
  if (q_out != q)
    MC_REQUIRE(!overlap(q_out, out_bytes, k, 2 * (T * k_stride + kn)) &&
                   !overlap(q_out, out_bytes, v, 2 * (T * v_stride + kn)),
               "%s: q_out overlaps k or v", name);
  MC_REQUIRE(ctx, "%s: null context", name);
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  const RopeParams P{q, k, v, q_stride, k_stride, v_stride, n_heads, n_kv_heads,
                     n_heads + n_kv_heads * (v ? 2 : 1), q_norm_w, k_norm_w, eps, positions,
                     reinterpret_cast<const unsigned long long*>(turns), rot_dim, interleaved,
                     q_out, q_out_stride, reinterpret_cast<const unsigned long long*>(slots),
                     k_cache, v_cache, num_blocks, block_size, block_stride, k_scale, v_scale,
                     status};
  const bool f8 = kv_dtype == MC_DTYPE_E4M3;
  if (head_dim == 64)
    return f8 ? launch_rope<64, true>(ctx, P, n_tokens) : launch_rope<64, false>(ctx, P, n_tokens);
  return f8 ? launch_rope<128, true>(ctx, P, n_tokens) : launch_rope<128, false>(ctx, P, n_tokens);
}
