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
// Tile. A warp takes 32 keys a step and multiplies on the tensor cores
// (m16n8k16, fp32 accumulators), K and V as stored: the k index of Q.K^T may
// be any order of the dimensions as long as Q uses the same, so a lane's 16
// contiguous bytes of a K row serve as its fragments of two k-steps (four of
// an e4m3 row); the n index of P.V may be any order too, so a lane's 16
// contiguous bytes of a V row are eight n-tiles, paired with the next key's
// by byte permutes.
//
// Memory. Every warp has a ring of steps in shared memory that its own lanes
// fill with 1-D bulk copies, one for each run of keys that lie together in a
// page (8 keys at most): deep enough that an SM has 60 KB and more in flight,
// and filled across the borders of pieces, so that the next item's keys
// arrive while the last one is joined. The 8-key parts of a step start 32
// bytes (mod 128) apart, and a lane takes its keys from the part lane % 4:
// the 4 rows x 2 chunks that a quarter-warp reads from V fall into different
// banks although whole rows are multiples of 128 bytes.
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
#include "mc_async.cuh"
#include "paged_split.cuh"

namespace {

constexpr int kMaxCtas = 512;
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
  unsigned long long wait_ns;
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

// Waits (every lane polls) for a stage's bytes; false after `limit_ns`.
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity,
                                          unsigned long long limit_ns) {
  if (mc_mbar_test(bar, parity)) return true;
  const unsigned long long t0 = mc_globaltimer();
  do {
    if (mc_mbar_test_sleep(bar, parity, 1000)) return true;
  } while (mc_globaltimer() - t0 < limit_ns);
  return false;
}

// Four e4m3 bytes -> two f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
      " cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

constexpr int kPart = 8;              // keys of a part
constexpr int kStep = 4 * kPart;      // keys a warp takes at once, one a lane
constexpr int kPerSm = 2;             // CTAs an SM holds at once

// Shape of the kernel for a head dimension and cache type: warps and ring
// depth fill the shared memory of two CTAs an SM.
template <int D, bool F8>
struct Shape {
  static constexpr int kRow = D * (F8 ? 1 : 2);          // bytes of a key's row
  static constexpr int kPartBytes = kPart * kRow + 32;
  static constexpr int kHalf = 4 * kPartBytes;           // K or V of a step
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kWarps = D == 128 && !F8 ? 3 : 4;
  static constexpr int kStages = D == 64 ? (F8 ? 5 : 3) : 2;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kUnit = kWarps * kStep;           // keys of a unit
  static constexpr int kORow = D + 4;                    // floats of a row in o
  static constexpr size_t kRingBytes = (size_t)kWarps * kStages * kStage;
  static constexpr size_t kOBytes = (size_t)kWarps * kHeads * kORow * sizeof(float);
  static constexpr size_t kSmem = kRingBytes + kOBytes;
  static_assert(kPerSm * (kSmem + 2048) <= 228 * 1024, "two CTAs an SM");
};

__device__ __forceinline__ uint32_t word(const uint4& u, int i) {
  return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
}

// First dimension of n-tile `nt` of P.V for column n (its result element);
// four n-tiles from a multiple of 4 on are consecutive dimensions.
template <int D, bool F8>
__device__ __forceinline__ int v_dim(int nt, int n) {
  if (F8) return (D / 8) * n + nt;
  return 64 * (nt / 8) + 8 * n + nt % 8;
}

// Folds (m2, l2) into a running maximum and sum.
__device__ __forceinline__ void fold(float& m, float& l, float m2, float l2) {
  const float top = fmaxf(m, m2), use = top == -INFINITY ? 0.0f : top;
  l = __fmaf_rn(l, ex2(m - use), ex2(m2 - use) * l2);
  m = top;
}

template <int D, bool F8>
__global__ void __launch_bounds__(Shape<D, F8>::kThreads, kPerSm)
paged_attention_kernel(const PaParams P) {
  using S = Shape<D, F8>;
  constexpr int kT = D / 8;              // n-tiles of P.V
  constexpr int kKLoads = S::kRow / 64;  // 16-byte loads of a lane's K row part
  constexpr int kVWords = S::kRow / 32;  // words of a lane's V row part
  extern __shared__ __align__(128) uint8_t ring_s[];
  float* o_s = reinterpret_cast<float*>(ring_s + S::kRingBytes);  // [warp][head][kORow]
  __shared__ __align__(8) uint64_t full_s[S::kWarps][S::kStages];
  __shared__ uint32_t live_s[S::kWarps][S::kStages];
  __shared__ float m_s[S::kWarps][kHeads], l_s[S::kWarps][kHeads];
  __shared__ long long sums_s[S::kWarps];
  __shared__ long long in_row_s;
  __shared__ int row_s;
  __shared__ uint32_t last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < S::kWarps * S::kStages) mc_mbar_init(&full_s[0][0] + tid, 1);
  mc_fence_barrier_init();
  mc_pdl_launch_dependents();
  mc_pdl_wait();
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
  auto units_of = [&](int r) { return ps_units(row_of(r), S::kUnit); };

  // ---- this CTA's range of units, and the row it starts in
  const int per = (P.rows + S::kThreads - 1) / S::kThreads;
  const int r_lo = min(tid * per, P.rows), r_hi = min(r_lo + per, P.rows);
  long long mine = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    mine += (long long)units_of(r) * P.items;
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
  for (int w = 0; w < S::kWarps; ++w) {
    if (w < warp) incl += sums_s[w];
    U += sums_s[w];
  }
  const int G = (int)min((long long)gridDim.x, U);
  if (cta >= G) return;
  const long long u0 = ps_begin(U, cta, G), u_end = ps_begin(U, cta + 1, G);
  if (u0 >= incl - mine && u0 < incl) {
    long long at = incl - mine;
    int r = r_lo;
    for (; r < r_hi - 1; ++r) {
      const long long n = (long long)units_of(r) * P.items;
      if (u0 < at + n) break;
      at += n;
    }
    row_s = r;
    in_row_s = u0 - at;
  }
  __syncthreads();

  // ---- filling the ring: the step at fill_base of the piece `fill`
  uint8_t* ring = ring_s + (size_t)warp * S::kStages * S::kStage;
  const uint64_t policy = mc_policy_evict_normal();
  PsCursor fill = ps_first(row_s, in_row_s, units_of(row_s), P.items, u_end - u0);
  PsCursor piece = fill;
  int fill_base = 0, fill_hi = 0, fill_head = 0, page = -1;
  uint32_t filled = 0;
  bool more = true;
  const int32_t* table = nullptr;
  auto enter = [&]() {  // the piece `fill`
    const PsRow keys = row_of(fill.row);
    const int lo = keys.low + fill.unit * S::kUnit;
    fill_hi = (int)min((long long)keys.len, (long long)lo + (long long)fill.units * S::kUnit);
    fill_base = lo + warp * kStep;
    fill_head = fill.item / P.subs;
    table = P.table + (size_t)(P.row_req ? max(P.row_req[fill.row], 0) : fill.row) * P.width;
  };
  // to the next step of this warp; its page numbers are on their way afterwards
  auto seek = [&]() {
    while (more && fill_base >= fill_hi) {
      more = ps_next(fill, P.items, P.rows, units_of);
      if (more) enter();
    }
    const int tok = fill_base + lane;
    page = more && tok < fill_hi ? table[tok / P.block_size] : -1;
  };
  auto issue = [&]() {
    const int stage = filled % S::kStages;
    const int tok = fill_base + lane, in_page = tok % P.block_size;
    const bool live = tok < fill_hi && page >= 0 && page < P.num_blocks;
    if (tok < fill_hi && !live && P.status) atomicOr(P.status, MC_KV_BAD_PAGE);
    const uint32_t all = __ballot_sync(0xffffffffu, live);
    uint64_t* bar = &full_s[warp][stage];
    if (lane == 0) {
      live_s[warp][stage] = all;
      mc_mbar_expect_tx(bar, 2 * S::kRow * __popc(all));
    }
    // a run starts a part, a page, or follows a key that is left out
    const bool starts =
        live && (lane % kPart == 0 || in_page == 0 || !((all >> (lane - 1)) & 1u));
    const uint32_t stops = __ballot_sync(0xffffffffu, starts || !live) >> lane >> 1;
    __syncwarp();
    if (starts) {
      const int n = min(stops ? __ffs(stops) : kPart, kPart - lane % kPart);
      const size_t off = ((size_t)page * P.block_stride +
                          ((size_t)fill_head * P.block_size + in_page) * D) * (F8 ? 1 : 2);
      uint8_t* to = ring + stage * S::kStage + lane / kPart * S::kPartBytes + lane % kPart * S::kRow;
      mc_bulk_g2s(to, static_cast<const uint8_t*>(P.kc) + off, n * S::kRow, bar, policy);
      mc_bulk_g2s(to + S::kHalf, static_cast<const uint8_t*>(P.vc) + off, n * S::kRow, bar, policy);
    }
    ++filled;
    fill_base += S::kUnit;
    seek();
  };
  enter();
  seek();
  for (int i = 0; i < S::kStages && more; ++i) issue();

  uint32_t used = 0;
  bool gave_up = false;
  const int c = lane & 3, hr = lane >> 2;
  do {
    const PsRow keys = row_of(piece.row);
    const int row = piece.row;
    const int kvh = piece.item / P.subs, sub = piece.item - kvh * P.subs;
    const int head0 = kvh * P.group + sub * kHeads, heads = min(kHeads, P.group - sub * kHeads);
    const int lo = keys.low + piece.unit * S::kUnit;
    const int hi = (int)min((long long)keys.len, (long long)lo + (long long)piece.units * S::kUnit);

    // ---- Q: row lane/4 of the tile (heads past the item's are zero)
    uint32_t qa[D / 16][2];
    float qk = P.scale_log2;
    {
      const uint16_t* q = P.q + (size_t)row * P.q_stride + (size_t)(head0 + hr) * D;
      if (!F8) {
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (hr < heads) w = __ldg(reinterpret_cast<const uint4*>(q) + c + 4 * i);
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
        for (int i = 0; i < kKLoads; ++i)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (hr < heads) w = __ldg(reinterpret_cast<const uint4*>(q) + 2 * c + 8 * i + z);
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

    for (int base = lo + warp * kStep; base < hi; base += S::kUnit) {
      const int stage = used % S::kStages;
      if (!wait_full(&full_s[warp][stage], (used / S::kStages) & 1, gave_up ? 0 : P.wait_ns)) {
        gave_up = true;  // nothing more is issued: the stage's barrier may still be open
        more = false;
        if (lane == 0 && P.status) atomicOr(P.status, MC_KV_WAIT);
      }
      const uint32_t live = live_s[warp][stage] >> (kPart * c) & 0xffu;
      const uint8_t* ks = ring + stage * S::kStage + (hr >> 1) * S::kPartBytes + (hr & 1) * S::kRow + 16 * c;
      const uint8_t* vs = ring + stage * S::kStage + S::kHalf + c * S::kPartBytes +
                          (F8 && D == 64 ? 8 : 16) * hr;
      // ---- scores of 32 keys for 8 heads; key 8 c + 4 z + 2 j + x in t[z][2 j + x]
      float t[2][4];
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < kKLoads; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(ks + (4 * z + 2 * j) * S::kRow + 64 * i);
            if (!F8) {
              mma16816<false>(s, qa[2 * i][0], 0u, qa[2 * i][1], 0u, w.x, w.y);
              mma16816<false>(s, qa[2 * i + 1][0], 0u, qa[2 * i + 1][1], 0u, w.z, w.w);
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                uint32_t b0, b1;
                e4m3x4_to_f16(word(w, x), b0, b1);
                mma16816<true>(s, qa[4 * i + x][0], 0u, qa[4 * i + x][1], 0u, b0, b1);
              }
            }
          }
          t[z][2 * j] = s[0] * qk;
          t[z][2 * j + 1] = s[1] * qk;
        }
      // ---- running maximum and sum of head lane/4
      if (live != 0xffu) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(live >> i & 1u)) t[i / 4][i % 4] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(t[0][0], t[0][1]), fmaxf(t[0][2], t[0][3])),
                        fmaxf(fmaxf(t[1][0], t[1][1]), fmaxf(t[1][2], t[1][3])));
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
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = ex2(t[z][i] - m_use);
          l += p[i];
        }
        const uint32_t h0 = pack2<F8>(p[0], p[1]), h1 = pack2<F8>(p[2], p[3]);
        const float2 g0 = unpack2<F8>(h0), g1 = unpack2<F8>(h1);
        const uint32_t w0 = pack2<F8>(p[0] - g0.x, p[1] - g0.y);
        const uint32_t w1 = pack2<F8>(p[2] - g1.x, p[3] - g1.y);
        uint32_t v[4][kVWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* vr = vs + (4 * z + i) * S::kRow;
          if (F8 && D == 64) {
            const uint2 u = *reinterpret_cast<const uint2*>(vr);
            v[i][0] = u.x;
            v[i][1] = u.y;
          } else {
#pragma unroll
            for (int n = 0; n < kVWords / 4; ++n) {
              const uint4 u = *reinterpret_cast<const uint4*>(vr + 128 * n);
              v[i][4 * n] = u.x;
              v[i][4 * n + 1] = u.y;
              v[i][4 * n + 2] = u.z;
              v[i][4 * n + 3] = u.w;
            }
          }
          // a key left out has a weight of zero, but what lies in its place may be NaN
          if (live != 0xffu && !(live >> (4 * z + i) & 1u)) {
#pragma unroll
            for (int n = 0; n < kVWords; ++n) v[i][n] = 0u;
          }
        }
        // ---- o += P V: rows 0-7 the high parts, rows 8-15 the low parts
        if (!F8) {
#pragma unroll
          for (int i = 0; i < kT / 2; ++i) {
            mma16816<false>(o[2 * i], h0, w0, h1, w1, __byte_perm(v[0][i], v[1][i], 0x5410),
                            __byte_perm(v[2][i], v[3][i], 0x5410));
            mma16816<false>(o[2 * i + 1], h0, w0, h1, w1, __byte_perm(v[0][i], v[1][i], 0x7632),
                            __byte_perm(v[2][i], v[3][i], 0x7632));
          }
        } else {
#pragma unroll
          for (int i = 0; i < kT / 4; ++i) {
            uint32_t b0[4], b1[4];
            e4m3x4_to_f16(__byte_perm(v[0][i], v[1][i], 0x5140), b0[0], b0[1]);
            e4m3x4_to_f16(__byte_perm(v[0][i], v[1][i], 0x7362), b0[2], b0[3]);
            e4m3x4_to_f16(__byte_perm(v[2][i], v[3][i], 0x5140), b1[0], b1[1]);
            e4m3x4_to_f16(__byte_perm(v[2][i], v[3][i], 0x7362), b1[2], b1[3]);
#pragma unroll
            for (int x = 0; x < 4; ++x)
              mma16816<true>(o[4 * i + x], h0, w0, h1, w1, b0[x], b1[x]);
          }
        }
      }
      ++used;
      __syncwarp();  // every lane has read the stage
      if (more) issue();
    }

    // ---- the warps' results of this piece
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (gave_up) l = __uint_as_float(0x7fc00000u);  // what did not arrive makes the result NaN
    __syncthreads();  // the piece before is done with the shared arrays
    if (c == 0) {
      m_s[warp][hr] = m;
      l_s[warp][hr] = l;
    }
#pragma unroll
    for (int i = 0; i < kT; i += 4)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float4*>(o_s + (warp * kHeads + hr) * S::kORow + v_dim<D, F8>(i, 2 * c + x)) =
            make_float4(o[i][x] + o[i][x + 2], o[i + 1][x] + o[i + 1][x + 2],
                        o[i + 2][x] + o[i + 2][x + 2], o[i + 3][x] + o[i + 3][x + 2]);
    __syncthreads();
    const bool begins = piece.unit == 0, ends = piece.unit + piece.units == piece.n;
    float* part = P.parts + part_floats(D) * (2 * (size_t)cta + (begins ? 1 : 0));
    auto finish = [&](int h, int d, float mx, float sum, float val) {
      if (h >= heads) return;
      const float vscale = F8 && P.v_scale ? P.v_scale[kvh] : 1.0f;
      const float r = sum == 0.0f ? 0.0f : __fdiv_rn(val, sum) * vscale;
      P.out[(size_t)row * P.out_stride + (size_t)(head0 + h) * D + d] = mc_f32_to_bf16(r);
      if (P.lse && d == 0)
        P.lse[(size_t)row * P.H + head0 + h] =
            sum == 0.0f ? -INFINITY : __fmaf_rn(mx, kLn2, logf(sum));
    };
    for (int i = tid; i < kHeads * D; i += S::kThreads) {
      const int h = i / D, d = i % D;
      float mx = m_s[0][h];
#pragma unroll
      for (int w = 1; w < S::kWarps; ++w) mx = fmaxf(mx, m_s[w][h]);
      const float use = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f, val = 0.0f;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const float a = ex2(m_s[w][h] - use);
        sum = __fmaf_rn(a, l_s[w][h], sum);
        val = __fmaf_rn(a, o_s[(w * kHeads + h) * S::kORow + d], val);
      }
      if (begins && ends) {
        finish(h, d, mx, sum, val);
      } else {
        part[i] = val;
        if (d == 0) {
          part[kHeads * D + h] = mx;
          part[kHeads * D + kHeads + h] = sum;
        }
      }
    }
    if (begins && ends) continue;
    // ---- the last of the item's CTAs joins the pieces in order
    const long long first_unit = u_end - piece.left - piece.unit;
    const int first_cta = begins ? cta : ps_owner(first_unit, U, G);
    const int last_cta = ends ? cta : ps_owner(first_unit + piece.n - 1, U, G);
    __threadfence();
    __syncthreads();
    if (tid == 0) {
      const uint32_t done = atomicAdd(P.counters + first_cta, 1u);
      last_s = done == (uint32_t)(last_cta - first_cta);
      if (last_s) P.counters[first_cta] = 0;
    }
    __syncthreads();
    if (!last_s) continue;
    __threadfence();
    auto part_of = [&](int x) {
      return P.parts + part_floats(D) * (2 * (size_t)x + (x == first_cta ? 1 : 0));
    };
    {  // the largest m and the sum, head tid % 8, pieces tid / 8, tid / 8 + threads / 8, ...
      const int h = tid % kHeads;
      float mx = -INFINITY, sum = 0.0f;
      for (int x = first_cta + tid / kHeads; x <= last_cta; x += S::kThreads / kHeads) {
        const float* pp = part_of(x) + kHeads * D + h;
        fold(mx, sum, __ldcg(pp), __ldcg(pp + kHeads));
      }
#pragma unroll
      for (int d = kHeads; d < 32; d <<= 1)
        fold(mx, sum, __shfl_xor_sync(0xffffffffu, mx, d), __shfl_xor_sync(0xffffffffu, sum, d));
      if (lane < kHeads) {
        m_s[warp][lane] = mx;
        l_s[warp][lane] = sum;
      }
    }
    __syncthreads();
    // four elements a thread, 8 pieces' loads in flight
    for (int i = tid; i < heads * D / 4; i += S::kThreads) {
      const int h = 4 * i / D;
      float mx = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w)
        fold(mx, sum, m_s[w][h], l_s[w][h]);
      const float use = mx == -INFINITY ? 0.0f : mx;
      float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int x0 = first_cta; x0 <= last_cta; x0 += 8) {
        float4 v[8];
        float m8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int x = x0 + k;
          m8[k] = -INFINITY;
          v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (x <= last_cta) {
            v[k] = __ldcg(reinterpret_cast<const float4*>(part_of(x)) + i);
            m8[k] = __ldcg(part_of(x) + kHeads * D + h);
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float a = ex2(m8[k] - use);
          val.x = __fmaf_rn(a, v[k].x, val.x);
          val.y = __fmaf_rn(a, v[k].y, val.y);
          val.z = __fmaf_rn(a, v[k].z, val.z);
          val.w = __fmaf_rn(a, v[k].w, val.w);
        }
      }
      const int d = 4 * i % D;
      finish(h, d, mx, sum, val.x);
      finish(h, d + 1, mx, sum, val.y);
      finish(h, d + 2, mx, sum, val.z);
      finish(h, d + 3, mx, sum, val.w);
    }
  } while (ps_next(piece, P.items, P.rows, units_of));
  if (gave_up) {  // copies still on their way end before the shared memory goes
    for (uint32_t i = filled > S::kStages ? filled - S::kStages : 0; i < filled; ++i)
      wait_full(&full_s[warp][i % S::kStages], (i / S::kStages) & 1, P.wait_ns);
  }
}

template <int D, bool F8>
int launch_attention(mc_ctx* ctx, const PaParams& P) {
  using S = Shape<D, F8>;
  auto fn = paged_attention_kernel<D, F8>;
  MC_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  long long g = (long long)ctx->num_sms * kPerSm;
  const long long most =
      (((long long)P.width * P.block_size + S::kUnit - 1) / S::kUnit) * P.rows * P.items;
  if (g > most) g = most;
  if (g > kMaxCtas) g = kMaxCtas;
  MC_CUDA(mc_launch_pdl(fn, dim3((unsigned)g), dim3(S::kThreads), S::kSmem, ctx->stream, P));
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
                   reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes), status,
                   mc_wait_limit(ctx, 1000000000ull)};
  const bool f8 = kv_dtype == MC_DTYPE_E4M3;
  if (head_dim == 64)
    return f8 ? launch_attention<64, true>(ctx, P) : launch_attention<64, false>(ctx, P);
  return f8 ? launch_attention<128, true>(ctx, P) : launch_attention<128, false>(ctx, P);
}
