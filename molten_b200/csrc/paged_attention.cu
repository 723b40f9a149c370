// Attention of new tokens over the paged cache (mc_paged_attention).
//
// For query row r and query head h with its KV head, over the row's keys j:
//   s_j = scale (q . k_j),  m = max s_j,  l = sum exp(s_j - m),
//   o = sum exp(s_j - m) v_j / l,  lse = m + log l
// in one pass over K and V with a running maximum and sum (each new maximum
// rescales what is summed so far), all sums in fp32; a row without keys gives
// zeros and lse = -inf.
//
// What bounds it: every K and V byte is read once and used by the group of
// query heads that share it (2 x group x 2 operations for each element), far
// below the tensor cores' rate: HBM bandwidth, and latency at short contexts.
//
// Tile. A warp takes 16 keys a step and multiplies on the tensor cores
// (m16n8k16, fp32 accumulators) straight from registers, with no shared
// memory: the k index of Q.K^T may be any order of the dimensions as long as
// Q uses the same, so a lane's 16 contiguous bytes of a K row serve as its
// fragments of two k-steps; the n index of P.V may be any order too, so a
// lane's 16 contiguous bytes of a V row are eight n-tiles, paired with the
// next token's by byte permutes. Each load instruction covers whole 64- or
// 128-byte parts of rows. The next step's 4 to 8 KB a warp are in flight
// while a step is computed.
//
// Rounding of P. Eight heads fill rows 0-7 of the 16-row tile; P is split
// into high and low parts (bf16 + bf16, or f16 + f16 for an e4m3 cache) and
// the low part rides in rows 8-15 at no cost, so P enters the product with
// 16 bits or more and the output's own rounding is the only one that counts.
// With an e4m3 cache K and V become f16 exactly, and Q becomes f16 scaled by
// a power of two a row (its largest value near 1), which loses nothing above
// 2^-24 of that value.
//
// Split. paged_split.cuh deals equal runs of keys to every CTA whatever the
// rows' lengths, so one long row fills the GPU and ragged batches balance.
// An item that spans CTAs leaves (m, l, o) of each piece in the workspace;
// the CTA that finishes last (an atomic count, nothing waits) joins them in
// piece order, so results do not depend on timing.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <math.h>

#include "kv_common.cuh"
#include "paged_split.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 16;               // keys a warp takes at once
constexpr int kUnit = kStep * kWarps;   // keys of a unit
constexpr int kMaxCtas = 1024;
constexpr int kHeads = 8;               // query heads of an item
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A piece's partial result in the workspace: o[8][D], m[8], l[8].
constexpr size_t part_floats(int D) { return (size_t)kHeads * D + 2 * kHeads; }
constexpr size_t kCounterBytes = kMaxCtas * sizeof(uint32_t);

struct PaParams {
  const uint16_t* q;
  size_t q_stride;
  int rows, H, K, group, subs, items;  // items of a row = K * subs
  const void* kc;
  const void* vc;
  int num_blocks, block_size;
  size_t block_stride;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int n_req, width;
  const int32_t* kv_lens;
  const int32_t* row_req;
  int window;
  float scale_log2;
  uint16_t* out;
  size_t out_stride;
  float* lse;
  uint32_t* counters;
  float* parts;
  uint32_t* status;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool F16>
__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two floats as a packed pair (a low, b high) and the pair's values back.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if (F16) {
    __half2 h;
    memcpy(&h, &u, 4);
    return __half22float2(h);
  }
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

// Four e4m3 bytes -> two f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
      " cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

__device__ __forceinline__ uint2 ldg_stream8(const void* p) {
  uint2 r;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(r.x), "=r"(r.y)
               : "l"(p));
  return r;
}

// Registers of one step: a lane's parts of two K rows (keys lane/4 and 8 +
// lane/4) and of four V rows (keys 2 (lane%4) + {0, 1, 8, 9}).
//
// K: a lane's 16-byte chunks lane%4 + 4i of the row; a chunk is `ks` k-steps.
// V: bf16 chunk i holds dims 64 i + 8 (lane/4) + e; e4m3 dims D/8 (lane/4) + e.
template <int D, bool F8>
struct Step {
  static constexpr int kRowBytes = D * (F8 ? 1 : 2);
  static constexpr int kKLoads = kRowBytes / 64;        // 16-byte loads a K row
  static constexpr int kVWords = kRowBytes / 32;        // 4-byte words a lane of a V row
  uint4 k[2][kKLoads];
  uint32_t v[4][kVWords];
  uint32_t live;  // bit i: V key i (and so score i) exists

  __device__ __forceinline__ void load(const PaParams& P, long long off, int lane) {
    const uint8_t* kc = static_cast<const uint8_t*>(P.kc);
    const uint8_t* vc = static_cast<const uint8_t*>(P.vc);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long long o = __shfl_sync(0xffffffffu, off, 8 * j + (lane >> 2));
#pragma unroll
      for (int i = 0; i < kKLoads; ++i) {
        k[j][i] = make_uint4(0, 0, 0, 0);
        if (o >= 0) k[j][i] = mc_ldg_stream(kc + o + 16 * ((lane & 3) + 4 * i));
      }
    }
    live = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long o =
          __shfl_sync(0xffffffffu, off, 2 * (lane & 3) + (i & 1) + 8 * (i >> 1));
      if (o >= 0) live |= 1u << i;
      if (F8 && D == 64) {
        uint2 u = make_uint2(0, 0);
        if (o >= 0) u = ldg_stream8(vc + o + 8 * (lane >> 2));
        v[i][0] = u.x;
        v[i][1] = u.y;
      } else {
#pragma unroll
        for (int n = 0; n < kVWords / 4; ++n) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (o >= 0) u = mc_ldg_stream(vc + o + 128 * n + 16 * (lane >> 2));
          v[i][4 * n] = u.x;
          v[i][4 * n + 1] = u.y;
          v[i][4 * n + 2] = u.z;
          v[i][4 * n + 3] = u.w;
        }
      }
    }
  }
};

__device__ __forceinline__ uint32_t word(const uint4& u, int i) {
  return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
}

// First dimension of n-tile `nt` of P.V for column n (its result element).
template <int D, bool F8>
__device__ __forceinline__ int v_dim(int nt, int n) {
  if (F8) return (D / 8) * n + nt;
  return 64 * (nt / 8) + 8 * n + nt % 8;
}

// CTAs an SM holds at once (the register bound the kernel is compiled to).
template <int D>
constexpr int kPerSm = D == 64 ? 3 : 2;

template <int D, bool F8>
__global__ void __launch_bounds__(kThreads, kPerSm<D>)
paged_attention_kernel(const PaParams P) {
  using S = Step<D, F8>;
  constexpr int kT = D / 8;  // n-tiles of P.V
  __shared__ float o_s[kWarps][kHeads][D];
  __shared__ float m_s[kWarps][kHeads], l_s[kWarps][kHeads];
  __shared__ long long sums_s[kWarps];
  __shared__ long long start_s;
  __shared__ int row_s;
  __shared__ uint32_t last_s;
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // keys the table can hold; key indices stay clear of the int range's end
  const long long capacity = min((long long)P.width * P.block_size, 0x7fff0000ll);
  const int cta = blockIdx.x;

  auto row_of = [&](int r) {
    int len = P.kv_lens[r];
    if (P.row_req) {
      const int req = P.row_req[r];
      if (req < 0 || req >= P.n_req) len = 0;
    }
    return ps_row(len, capacity, P.window);
  };

  // ---- this CTA's range of units, and the row it starts in
  const int per = (P.rows + kThreads - 1) / kThreads;
  const int r_lo = min(tid * per, P.rows), r_hi = min(r_lo + per, P.rows);
  long long mine = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    mine += (long long)ps_units(row_of(r), kUnit) * P.items;
    if (cta == 0 && P.status) {
      if (P.kv_lens[r] < 0 || P.kv_lens[r] > capacity) atomicOr(P.status, MC_KV_BAD_LENGTH);
      if (P.row_req && (P.row_req[r] < -1 || P.row_req[r] >= P.n_req))
        atomicOr(P.status, MC_KV_BAD_ROW);
    }
  }
  long long incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) sums_s[warp] = incl;
  __syncthreads();
  long long U = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) incl += sums_s[w];
    U += sums_s[w];
  }
  const int G = (int)min((long long)gridDim.x, U);
  if (cta >= G) return;
  long long u = ps_begin(U, cta, G);
  const long long u_end = ps_begin(U, cta + 1, G);
  if (u >= incl - mine && u < incl) {
    long long at = incl - mine;
    int r = r_lo;
    for (;; ++r) {
      const long long n = (long long)ps_units(row_of(r), kUnit) * P.items;
      if (u < at + n) break;
      at += n;
    }
    row_s = r;
    start_s = at;
  }
  __syncthreads();
  int row = row_s;
  long long row_start = start_s;

  while (u < u_end) {
    const PsRow keys = row_of(row);
    const int n = ps_units(keys, kUnit);
    if (u >= row_start + (long long)n * P.items) {
      row_start += (long long)n * P.items;
      ++row;
      continue;
    }
    const PsPiece piece = ps_piece(u, u_end, row, row_start, n, U, G);
    u += piece.units;
    const int kvh = piece.item / P.subs, head0 = kvh * P.group + (piece.item % P.subs) * kHeads;
    const int heads = min(kHeads, P.group - (piece.item % P.subs) * kHeads);
    const int lo = keys.low + piece.unit * kUnit;
    const int hi = (int)min((long long)keys.len, (long long)lo + (long long)piece.units * kUnit);
    const int32_t* table = P.table + (size_t)(P.row_req ? max(P.row_req[row], 0) : row) * P.width;

    // byte offset of the key this lane (0..15) looks up, -1: none
    auto look = [&](int base) -> long long {
      const int tok = base + lane;
      if (lane >= kStep || tok >= hi) return -1;
      const int b = tok / P.block_size;
      const int page = table[b];
      if (page < 0 || page >= P.num_blocks) {
        if (P.status) atomicOr(P.status, MC_KV_BAD_PAGE);
        return -1;
      }
      return ((long long)page * (long long)P.block_stride +
              ((long long)kvh * P.block_size + (tok - b * P.block_size)) * D) *
             (F8 ? 1 : 2);
    };

    // ---- Q: row lane/4 of the tile (heads past the item's are zero)
    const int hr = lane >> 2;
    uint32_t qa[D / 16][2];
    float qk = P.scale_log2;
    {
      const uint16_t* q = P.q + (size_t)row * P.q_stride + (size_t)(head0 + hr) * D;
      if (!F8) {
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (hr < heads) w = __ldg(reinterpret_cast<const uint4*>(q) + (lane & 3) + 4 * i);
          qa[2 * i][0] = w.x;
          qa[2 * i][1] = w.y;
          qa[2 * i + 1][0] = w.z;
          qa[2 * i + 1][1] = w.w;
        }
      } else {
        // dims 16 (lane%4) + 64 i + 0..15: two 16-byte loads for each K load
        float f[D / 4];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (hr < heads) w = __ldg(reinterpret_cast<const uint4*>(q) + 2 * (lane & 3) + 8 * i + z);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float2 p = unpack2<false>(word(w, x));
              f[16 * i + 8 * z + 2 * x] = p.x;
              f[16 * i + 8 * z + 2 * x + 1] = p.y;
              top = fmaxf(top, fmaxf(fabsf(p.x), fabsf(p.y)));
            }
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e with 2^e <= top < 2^(e+1); 1 for zero, subnormal or infinite rows
        const int e = (int)(__float_as_uint(top) >> 23) - 127;
        const bool plain = e < -126 || e > 126;
        const float down = plain ? 1.0f : __uint_as_float((uint32_t)(127 - e) << 23);
        const float up = plain ? 1.0f : __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            qa[i][x] = pack2<true>(f[4 * i + 2 * x] * down, f[4 * i + 2 * x + 1] * down);
        qk *= up;
        if (P.k_scale) qk *= P.k_scale[kvh];
      }
    }

    float o[kT][4];
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    int base = lo + warp * kStep;
    S cur, nxt;
    if (base < hi) cur.load(P, look(base), lane);
    long long off = look(base + kUnit);
    for (; base < hi; base += kUnit) {
      if (base + kUnit < hi) nxt.load(P, off, lane);
      off = look(base + 2 * kUnit);
      // ---- scores of 2 x 8 keys for 8 heads
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
#pragma unroll
        for (int i = 0; i < S::kKLoads; ++i) {
          const uint4 w = cur.k[j][i];
          if (!F8) {
            mma16816<false>(s[j], qa[2 * i][0], 0u, qa[2 * i][1], 0u, w.x, w.y);
            mma16816<false>(s[j], qa[2 * i + 1][0], 0u, qa[2 * i + 1][1], 0u, w.z, w.w);
          } else {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t b0, b1;
              e4m3x4_to_f16(word(w, x), b0, b1);
              mma16816<true>(s[j], qa[4 * i + x][0], 0u, qa[4 * i + x][1], 0u, b0, b1);
            }
          }
        }
      }
      // ---- running maximum and sum of head lane/4
      float t[4] = {s[0][0] * qk, s[0][1] * qk, s[1][0] * qk, s[1][1] * qk};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(cur.live >> i & 1)) t[i] = -INFINITY;
      float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float m_new = fmaxf(m, top);
      const float m_use = m_new == -INFINITY ? 0.0f : m_new;
      if (__any_sync(0xffffffffu, m_new != m)) {
        const float a = ex2(m - m_use);
        l *= a;
#pragma unroll
        for (int i = 0; i < kT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][x] *= a;
        m = m_new;
      }
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = ex2(t[i] - m_use);
        l += p[i];
      }
      const uint32_t h0 = pack2<F8>(p[0], p[1]), h1 = pack2<F8>(p[2], p[3]);
      const float2 g0 = unpack2<F8>(h0), g1 = unpack2<F8>(h1);
      const uint32_t w0 = pack2<F8>(p[0] - g0.x, p[1] - g0.y);
      const uint32_t w1 = pack2<F8>(p[2] - g1.x, p[3] - g1.y);
      // ---- o += P V: rows 0-7 the high parts, rows 8-15 the low parts
      if (!F8) {
#pragma unroll
        for (int i = 0; i < kT / 2; ++i) {
          mma16816<false>(o[2 * i], h0, w0, h1, w1, __byte_perm(cur.v[0][i], cur.v[1][i], 0x5410),
                          __byte_perm(cur.v[2][i], cur.v[3][i], 0x5410));
          mma16816<false>(o[2 * i + 1], h0, w0, h1, w1,
                          __byte_perm(cur.v[0][i], cur.v[1][i], 0x7632),
                          __byte_perm(cur.v[2][i], cur.v[3][i], 0x7632));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kT / 4; ++i) {
          uint32_t b0[4], b1[4];
          e4m3x4_to_f16(__byte_perm(cur.v[0][i], cur.v[1][i], 0x5140), b0[0], b0[1]);
          e4m3x4_to_f16(__byte_perm(cur.v[0][i], cur.v[1][i], 0x7362), b0[2], b0[3]);
          e4m3x4_to_f16(__byte_perm(cur.v[2][i], cur.v[3][i], 0x5140), b1[0], b1[1]);
          e4m3x4_to_f16(__byte_perm(cur.v[2][i], cur.v[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            mma16816<true>(o[4 * i + x], h0, w0, h1, w1, b0[x], b1[x]);
        }
      }
      cur = nxt;
    }

    // ---- the warps' results of this piece
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();  // the piece before is done with the shared arrays
    if ((lane & 3) == 0) {
      m_s[warp][hr] = m;
      l_s[warp][hr] = l;
    }
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        o_s[warp][hr][v_dim<D, F8>(i, 2 * (lane & 3) + x)] = o[i][x] + o[i][x + 2];
    __syncthreads();
    const bool whole = piece.first_cta == piece.last_cta;
    float* part = P.parts + part_floats(D) * (2 * (size_t)cta + (cta == piece.first_cta ? 1 : 0));
    auto finish = [&](int h, int d, float mx, float sum, float val) {
      if (h >= heads) return;
      const float vs = F8 && P.v_scale ? P.v_scale[kvh] : 1.0f;
      const float r = sum == 0.0f ? 0.0f : __fdiv_rn(val, sum) * vs;
      P.out[(size_t)row * P.out_stride + (size_t)(head0 + h) * D + d] = mc_f32_to_bf16(r);
      if (P.lse && d == 0)
        P.lse[(size_t)row * P.H + head0 + h] =
            sum == 0.0f ? -INFINITY : __fmaf_rn(mx, kLn2, logf(sum));
    };
    for (int i = tid; i < kHeads * D; i += kThreads) {
      const int h = i / D, d = i % D;
      float mx = m_s[0][h];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, m_s[w][h]);
      const float use = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f, val = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float a = ex2(m_s[w][h] - use);
        sum = __fmaf_rn(a, l_s[w][h], sum);
        val = __fmaf_rn(a, o_s[w][h][d], val);
      }
      if (whole) {
        finish(h, d, mx, sum, val);
      } else {
        part[i] = val;
        if (d == 0) {
          part[kHeads * D + h] = mx;
          part[kHeads * D + kHeads + h] = sum;
        }
      }
    }
    if (whole) continue;
    // ---- the last of the item's CTAs joins the pieces in order
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const uint32_t pieces = (uint32_t)(piece.last_cta - piece.first_cta + 1);
      const uint32_t done = atomicAdd(P.counters + piece.first_cta, 1u);
      last_s = done == pieces - 1;
      if (last_s) P.counters[piece.first_cta] = 0;
    }
    __syncthreads();
    if (!last_s) continue;
    __threadfence();
    for (int i = tid; i < kHeads * D; i += kThreads) {
      const int h = i / D, d = i % D;
      float mx = -INFINITY, sum = 0.0f, val = 0.0f;
      for (int c = piece.first_cta; c <= piece.last_cta; ++c) {
        const float* pp = P.parts + part_floats(D) * (2 * (size_t)c + (c == piece.first_cta ? 1 : 0));
        const float mc = __ldcg(pp + kHeads * D + h);
        const float m2 = fmaxf(mx, mc);
        const float use = m2 == -INFINITY ? 0.0f : m2;
        const float a = ex2(mx - use), b = ex2(mc - use);
        sum = __fmaf_rn(sum, a, b * __ldcg(pp + kHeads * D + kHeads + h));
        val = __fmaf_rn(val, a, b * __ldcg(pp + i));
        mx = m2;
      }
      finish(h, d, mx, sum, val);
    }
  }
}

template <int D, bool F8>
int launch_attention(mc_ctx* ctx, const PaParams& P) {
  long long g = (long long)ctx->num_sms * kPerSm<D>;
  const long long most = (((long long)P.width * P.block_size + kUnit - 1) / kUnit) * P.rows * P.items;
  if (g > most) g = most;
  if (g > kMaxCtas) g = kMaxCtas;
  MC_CUDA(mc_launch_pdl(paged_attention_kernel<D, F8>, dim3((unsigned)g), dim3(kThreads), 0,
                        ctx->stream, P));
  return mc_after_launch("paged_attention_kernel");
}

}  // namespace

extern "C" size_t mc_paged_attention_workspace_bytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  return kCounterBytes + 2 * (size_t)kMaxCtas * part_floats(head_dim) * sizeof(float);
}

extern "C" int mc_paged_attention(mc_ctx* ctx, const uint16_t* q, size_t q_stride, int n_rows,
                                  int n_heads, const void* k_cache, const void* v_cache,
                                  int kv_dtype, int num_blocks, int block_size,
                                  size_t block_stride, int n_kv_heads, int head_dim,
                                  const float* k_scale, const float* v_scale,
                                  const int32_t* block_table, int n_req, int table_width,
                                  const int32_t* kv_lens, const int32_t* row_req, int window,
                                  float scale, uint16_t* out, size_t out_stride, float* lse,
                                  void* workspace, size_t ws_bytes, uint32_t* status) {
  const char* name = "paged_attention";
  int rc = mc_check_kv_cache(name, k_cache, v_cache, kv_dtype, num_blocks, block_size,
                             block_stride, n_kv_heads, head_dim, k_scale, v_scale);
  if (rc) return rc;
  MC_REQUIRE(n_rows >= 0, "%s: n_rows %d", name, n_rows);
  if (n_rows == 0) return MC_OK;
  MC_REQUIRE(n_heads >= 1 && n_heads <= 16384 && n_heads % n_kv_heads == 0,
             "%s: %d query heads for %d KV heads", name, n_heads, n_kv_heads);
  MC_REQUIRE(n_req >= 1 && table_width >= 1, "%s: block table [%d][%d]", name, n_req, table_width);
  MC_REQUIRE(row_req || n_rows <= n_req, "%s: %d rows for a block table of %d (row_req is null)",
             name, n_rows, n_req);
  MC_REQUIRE(window >= 0, "%s: window %d", name, window);
  MC_REQUIRE(isfinite(scale), "%s: scale must be finite", name);
  MC_REQUIRE(q && out && block_table && kv_lens && workspace, "%s: null pointer", name);
  MC_REQUIRE(mc_aligned(q, 16) && mc_aligned(out, 16), "%s: rows must be 16-byte aligned", name);
  const size_t qn = (size_t)n_heads * head_dim, far = (size_t)1 << 40;
  MC_REQUIRE(q_stride % 8 == 0 && out_stride % 8 == 0 && q_stride <= far && out_stride <= far,
             "%s: row strides must be multiples of 8 elements", name);
  MC_REQUIRE(n_rows <= 1 || out_stride >= qn, "%s: out rows overlap", name);
  MC_REQUIRE(mc_aligned(workspace, 16), "%s: workspace must be 16-byte aligned", name);
  MC_REQUIRE(ws_bytes >= mc_paged_attention_workspace_bytes(head_dim),
             "%s: workspace of %zu bytes, %zu needed", name, ws_bytes,
             mc_paged_attention_workspace_bytes(head_dim));
  // a query row is read by every CTA that holds a part of it while others write
  const uintptr_t a = (uintptr_t)q, b = (uintptr_t)out;
  const size_t q_bytes = 2 * ((size_t)(n_rows - 1) * q_stride + qn);
  const size_t o_bytes = 2 * ((size_t)(n_rows - 1) * out_stride + qn);
  MC_REQUIRE(a + q_bytes <= b || b + o_bytes <= a, "%s: out overlaps q", name);
  MC_REQUIRE(ctx, "%s: null context", name);
  McDeviceGuard dev(ctx->device);
  MC_CUDA(dev.error());
  const int group = n_heads / n_kv_heads, subs = (group + kHeads - 1) / kHeads;
  const PaParams P{q, q_stride, n_rows, n_heads, n_kv_heads, group, subs, n_kv_heads * subs,
                   k_cache, v_cache, num_blocks, block_size, block_stride, k_scale, v_scale,
                   block_table, n_req, table_width, kv_lens, row_req, window, scale * kLog2e, out,
                   out_stride, lse, static_cast<uint32_t*>(workspace),
                   reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes), status};
  const bool f8 = kv_dtype == MC_DTYPE_E4M3;
  if (head_dim == 64)
    return f8 ? launch_attention<64, true>(ctx, P) : launch_attention<64, false>(ctx, P);
  return f8 ? launch_attention<128, true>(ctx, P) : launch_attention<128, false>(ctx, P);
}
