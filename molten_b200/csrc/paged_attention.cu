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
// fill with 16-byte asynchronous copies, deep enough that an SM has 60 KB and
// more on their way, and filled across the borders of pieces, so that the next
// item's keys arrive while the last one is joined. (An earlier form of this
// kernel filled the ring by 1-D bulk copies, one for each run of keys that lie
// together in a page. When the two were compared they took as long for pages
// of 16 keys and up, bulk copies 14% longer for e4m3 rows of 64 bytes and 1.7
// times as long for pages of one key: a copy cost an SM some 47 cycles
// whatever its size.)
//
// Rounding of P. P is split into high and low parts (bf16 + bf16, or f16 + f16
// for an e4m3 cache), so it enters the product with 16 bits or more and the
// output's own rounding is the only one that counts. f16's last step is 2^-24:
// for an e4m3 cache the running maximum is taken 15 powers of two lower, so
// that the largest weight is 2^15, and weights have 16 bits down to 2^-24 of
// the largest one of the warp's keys, fewer below, and none below 2^-40 (with
// a largest weight of 1 a key of weight 2^-25 counted nothing, and one that
// outweighs a long flat tail but has V near zero left a result that was off by
// its own size). Eight heads fill rows 0-7 of the 16-row tile, and the low
// parts ride in rows 8-15 at no cost; where more than 8 heads share a KV head a tile takes 16 and the low parts cost
// products of their own (16 heads a KV head, 64 rows of 4000 to 8200 keys of
// 128: 464 us by eights, 245 us by sixteens, e4m3 273 and 172; of 64: 247 and
// 129, e4m3 161 and 116).
// With an e4m3 cache K and V become f16 exactly, and Q becomes f16 scaled by
// a power of two a row (its largest value near 1), which loses nothing above
// 2^-24 of that value.
//
// Split. paged_split.cuh deals equal runs of keys to every CTA whatever the
// rows' lengths, so one long row fills the GPU and ragged batches balance. One
// wave of CTAs: two or three times as many for the hardware to balance cost
// more in starts and joins than the uneven SMs do (131071 keys 52 -> 62, 64 us).
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
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The weights of an e4m3 cache's keys are 2^kUp times exp(s - max s), the most that f16 holds.
constexpr float kUp = 15.0f, kDown = 0x1p-15f;

// A piece's partial result in the workspace: o[heads][D], m[heads], l[heads] (8 or 16 heads).
constexpr size_t part_floats(int D, int heads) { return (size_t)heads * D + 2 * heads; }
constexpr size_t kCounterBytes = kMaxCtas * sizeof(uint32_t);

struct PaParams {
  const uint16_t* q;
  size_t q_stride;
  int rows, H, K, group, subs, items;  // items of a row = K * subs
  const void* kc;
  const void* vc;
  int num_blocks, block_size;
  uint32_t page_rows;  // block_stride / D
  PsDiv by_block;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  int n_req, width;
  int capacity;    // keys the table can hold, clear of the int range's end
  int small_unit;  // ps_small_unit
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
  int skip_arrive;  // test aids (mc_set_test_flags): a warp's copies are never reported as arrived
                    // (1), or by a lane that has given up on them (2)
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

// Waits (every lane polls) for a stage's bytes. False, for the whole warp alike, if any lane's wait
// ran past `limit_ns`: what follows takes all lanes together. A lane with `late` (a test's) gives up
// at once and reports then what the other lanes wait for.
__device__ __forceinline__ bool wait_full(uint64_t* bar, uint32_t parity, unsigned long long limit_ns,
                                          bool late) {
  bool ok = mc_mbar_test(bar, parity);
  if (__all_sync(0xffffffffu, ok)) return true;
  if (!ok) {
    const unsigned long long t0 = mc_globaltimer();
    const unsigned long long limit = late ? 0 : limit_ns;
    for (;;) {
      ok = mc_mbar_test_sleep(bar, parity, limit < 1000 ? (uint32_t)limit : 1000);
      if (ok) break;
      if (mc_globaltimer() - t0 >= limit) {
        if (late) mc_mbar_arrive(bar);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// Four e4m3 bytes -> two f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
      " cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

// Shape of the kernel for a head dimension and cache type: 8 warps an SM with
// rings that hold 128 to 192 KB, except e4m3 rows of 64 bytes, whose time goes
// into instructions more than into bytes and which take 12 warps (64 rows of
// 4000 to 8200 keys: 100 us with 8, 86 with 12; 131071 keys 43.4 and 39.3).
// bf16 rows of 64 at 12 warps and two steps a ring: 131071 keys 51.4 -> 50.4
// us, 32 rows of 17 to 6000 keys 40.8 -> 39.0, 64 rows of 4000 to 8200 keys
// 126.1 -> 127.1. Rows of 256 bytes take 16 keys a step, so that 4 warps' rings
// fit twice (131071 keys: 99.6 us with 32 keys a step and one CTA an SM, 90.9
// with 16 and two; 64 rows of 4000 to 8200 keys 257 and 239).
//
// A step's K, and its V, are 128-byte lines of 8 chunks (16 bytes; chunk ch of
// key k is number k kChunks + ch). A line's chunks are permuted, number n at
// n ^ turn with turn = 2 (k / kPart), ^ 4 for an odd key if a row is whole
// lines, so that the 8 chunks a quarter-warp reads at once (2 keys x 4 chunks
// of K, 4 parts x 2 chunks of V) fall into different banks.
template <int D, bool F8, int HEADS>
struct Shape {
  static constexpr int kHeads = HEADS;            // query heads of an item: 8 or 16
  static constexpr int kRow = D * (F8 ? 1 : 2);   // bytes of a key's row
  static constexpr int kChunks = kRow / 16;       // 16-byte chunks of a row
  static constexpr int kStep = kRow == 256 ? 16 : 32;  // keys a warp takes at once, one a lane
  static constexpr int kPart = kStep / 4;         // keys a lane's V fragments come from
  static constexpr int kHalf = kStep * kRow;      // K or V of a step
  static constexpr int kStage = 2 * kHalf;
  static constexpr int kWarps = 4;
  static constexpr int kStages = kRow == 64 ? 4 : D == 64 && HEADS == 8 ? 3 : 2;
  static constexpr int kPerSm = kRow == 64 && HEADS == 8 ? 3 : 2;  // CTAs an SM holds at once
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kUnit = kWarps * kStep;    // keys of a (small) unit
  static constexpr int kORow = D + 4;             // floats of a row in o
  static constexpr size_t kRingBytes = (size_t)kWarps * kStages * kStage;
  static constexpr size_t kOBytes = (size_t)kWarps * kHeads * kORow * sizeof(float);
  static constexpr size_t kSmem = kRingBytes + kOBytes;
  // a CTA has some 0.5 KB of static shared memory too, and the system takes 1 KB of each
  static_assert(kPerSm * (kSmem + 1536) <= 228 * 1024, "shared memory");
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

template <int D, bool F8, int HEADS>
__global__ void __launch_bounds__(Shape<D, F8, HEADS>::kThreads, (Shape<D, F8, HEADS>::kPerSm))
paged_attention_kernel(const PaParams P) {
  using S = Shape<D, F8, HEADS>;
  constexpr int kHeads = HEADS, kM = HEADS / 8;  // kM: heads lane/4 and, of 16, 8 + lane/4
  constexpr int kT = D / 8;              // n-tiles of P.V
  constexpr int kZ = S::kStep / 16;
  constexpr uint32_t kAll = (1u << S::kPart) - 1;
  constexpr int kKLoads = S::kRow / 64;  // 16-byte loads of a lane's K row part
  constexpr int kVWords = S::kRow / 32;  // words of a lane's V row part
  extern __shared__ __align__(128) uint8_t ring_s[];
  float* o_s = reinterpret_cast<float*>(ring_s + S::kRingBytes);  // [warp][head][kORow]
  __shared__ __align__(8) uint64_t full_s[S::kWarps][S::kStages];
  __shared__ uint32_t live_s[S::kWarps][S::kStages];
  __shared__ float m_s[S::kWarps][kHeads], l_s[S::kWarps][kHeads];
  __shared__ uint32_t last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a warp's own barriers, an arrival a lane (of 33 the last never comes, or late: a test's wait
  // that runs out)
  if (lane < S::kStages)
    mc_mbar_init(&full_s[warp][lane], P.skip_arrive && blockIdx.x == 0 && warp == 0 ? 33 : 32);
  mc_fence_barrier_init();
  __syncwarp();
  mc_pdl_launch_dependents();
  mc_pdl_wait();
  const int capacity = P.capacity;
  const int cta = blockIdx.x;

  auto row_of = [&](int r, int* of = nullptr) {
    int len = P.kv_lens[r], req = r;
    if (P.row_req) {
      req = P.row_req[r];
      if (req < 0 || req >= P.n_req) len = req = 0;
    }
    if (of) *of = req;
    return ps_row(len, capacity, P.window);
  };
  int unit = P.small_unit;  // keys of a unit
  auto units_of = [&](int r) { return ps_units(row_of(r), unit); };

  // ---- this CTA's range of units, and the row it starts in. Every warp finds them for itself:
  // a run of rows a lane, no barrier.
  const int per = (P.rows + 31) / 32;
  const int r_lo = min(lane * per, P.rows), r_hi = min(r_lo + per, P.rows);
  int mine, incl, U;  // units of this lane's rows, up to and with them, of all rows
  int n_max;
  auto scan = [&]() {
    mine = 0;
    n_max = 0;
    for (int r = r_lo; r < r_hi; ++r) {
      const int n = units_of(r);
      mine += n * P.items;
      n_max = max(n_max, n);
    }
    incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    U = __shfl_sync(0xffffffffu, incl, 31);
    n_max = __reduce_max_sync(0xffffffffu, n_max);
  };
  scan();
  const int factor = ps_factor(U, n_max, P.rows * P.items, gridDim.x);
  if (factor > 1) {
    unit = (int)min((long long)unit * factor, 0x7fffffffll);
    scan();
  }
  if (cta == 0 && warp == 0 && P.status)
    for (int r = r_lo; r < r_hi; ++r) {
      if (P.kv_lens[r] < 0 || P.kv_lens[r] > capacity) atomicOr(P.status, MC_KV_BAD_LENGTH);
      if (P.row_req && (P.row_req[r] < -1 || P.row_req[r] >= P.n_req))
        atomicOr(P.status, MC_KV_BAD_ROW);
    }
  const int cost = ps_cost(U, factor, gridDim.x);
  mine += cost * P.items * (r_hi - r_lo);
  incl += cost * P.items * r_hi;
  U += cost * P.items * P.rows;
  const int G = min((int)gridDim.x, U);
  if (cta >= G) return;
  const int u0 = ps_begin(U, cta, G), u_end = ps_begin(U, cta + 1, G);
  int row_at = incl - mine;
  int row0 = r_lo;
  const bool here = u0 >= row_at && u0 < incl;
  if (here) {
    for (; row0 < r_hi - 1; ++row0) {
      const int n = (units_of(row0) + cost) * P.items;
      if (u0 < row_at + n) break;
      row_at += n;
    }
  }
  const int owner = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
  row0 = __shfl_sync(0xffffffffu, row0, owner);
  row_at = __shfl_sync(0xffffffffu, row_at, owner);

  // ---- filling the ring: the step at fill_base of the piece `fill`
  uint8_t* ring = ring_s + (size_t)warp * S::kStages * S::kStage;
  PsCursor fill = ps_first(row0, u0 - row_at, units_of(row0), P.items, u_end - u0, cost);
  if (fill.units <= 0) return;  // no more than an item's start
  PsCursor piece = fill;
  int fill_base = 0, fill_hi = 0, fill_stage = 0, page = -1;
  uint32_t in_page = 0, head_row = 0;
  bool more = true;
  const int32_t* table = nullptr;
  auto enter = [&]() {  // the piece `fill`
    int req;  // read once: a table row that is there, whatever changes meanwhile
    const PsRow keys = row_of(fill.row, &req);
    const int lo = keys.low + fill.unit * unit;
    fill_hi = (int)min((long long)keys.len, (long long)lo + (long long)fill.units * unit);
    fill_base = lo + warp * S::kStep;
    head_row = (uint32_t)(fill.item / P.subs) * P.block_size;
    table = P.table + (size_t)req * P.width;
  };
  // to the next step of this warp; its page numbers are on their way afterwards
  auto seek = [&]() {
    while (more && fill_base >= fill_hi) {
      more = ps_next(fill, P.items, P.rows, units_of);
      if (more) enter();
    }
    const int tok = fill_base + lane;
    page = -1;
    if (more && lane < S::kStep && tok < fill_hi) {
      const int b = ps_div(tok, P.by_block);
      in_page = (uint32_t)(tok - b * P.block_size);
      page = table[b];
    }
  };
  // this lane copies chunk number lane + 32 i of the step, key i kKeys + lane / kChunks
  constexpr int kKeys = 32 / S::kChunks;
  const uint8_t* kc = static_cast<const uint8_t*>(P.kc) + 16 * (lane % S::kChunks);
  const uint8_t* vc = static_cast<const uint8_t*>(P.vc) + 16 * (lane % S::kChunks);
  auto issue = [&]() {
    const int tok = fill_base + lane;
    const bool there = lane < S::kStep && tok < fill_hi;
    const bool live = there && page >= 0 && page < P.num_blocks;
    if (there && !live && P.status) atomicOr(P.status, MC_KV_BAD_PAGE);
    const uint32_t all = __ballot_sync(0xffffffffu, live);
    if (lane == 0) live_s[warp][fill_stage] = all;
    const uint32_t row = live ? (uint32_t)page * P.page_rows + head_row + in_page : 0xffffffffu;
    uint8_t* to = ring + fill_stage * S::kStage;
    const int odd = S::kChunks >= 8 ? 4 * ((lane / S::kChunks) & 1) : 0;
#pragma unroll
    for (int i = 0; i < S::kStep / kKeys; ++i) {
      const int key = i * kKeys + lane / S::kChunks;
      const uint32_t r = __shfl_sync(0xffffffffu, row, key);
      const int turn = 2 * (key / S::kPart) ^ odd;
      const int at = 512 * i + 16 * (lane ^ turn);
      if (r != 0xffffffffu) {
        mc_cp_async16(to + at, kc + (size_t)r * S::kRow);
        mc_cp_async16(to + S::kHalf + at, vc + (size_t)r * S::kRow);
      }
    }
    mc_cp_async_arrive(&full_s[warp][fill_stage]);
    fill_stage = fill_stage + 1 == S::kStages ? 0 : fill_stage + 1;
    fill_base += S::kUnit;
    seek();
  };
  enter();
  seek();
  for (int i = 0; i < S::kStages && more; ++i) issue();
  __syncwarp();  // live_s of the first steps

  int stage = 0;
  uint32_t phase = 0;
  bool gave_up = false;
  const int c = lane & 3, hr = lane >> 2;
  // Where this lane reads: K key kPart (hr / 2) + hr % 2 (+ 4 z + 2 j), chunk c (+ 4 i: the other
  // half of the line for odd i); V key kPart c (+ 4 z + i), chunk hr (+ 8 n), or half a chunk.
  constexpr bool kHalfChunk = F8 && D == 64;
  const int k_turn = 16 * (c ^ (2 * (hr >> 1)) ^ (S::kChunks >= 8 ? 4 * (hr & 1) : 0));
  const int k_at = S::kChunks >= 8 ? (S::kPart * (hr >> 1) + (hr & 1)) * S::kRow + k_turn
                                   : (S::kPart * (hr >> 1)) * S::kRow + (k_turn ^ (64 * (hr & 1)));
  const int k_flip = (k_at ^ 64) - k_at;
  const int v_at = S::kPart * c * S::kRow +
                   (kHalfChunk ? 16 * ((hr >> 1) ^ (2 * c)) + 8 * (hr & 1) : 16 * (hr ^ (2 * c)));
  const int v_flip = (v_at ^ 64) - v_at;
  // Four elements of an item's result (quad `at`: head 4 at / D of the item) from their sums.
  auto finish = [&](int row, int head0, float vscale, int at, float mx, float sum, float4 v) {
    if (F8) {
      mx += kUp;
      sum *= kDown;
      v = make_float4(v.x * kDown, v.y * kDown, v.z * kDown, v.w * kDown);
    }
    const int head = head0 + 4 * at / D, d = 4 * at % D;
    const float by = sum == 0.0f ? 0.0f : __fdiv_rn(vscale, sum);  // NaN of a zero sum: 0
    uint2 r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.x) : "f"(v.y * by), "f"(v.x * by));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r.y) : "f"(v.w * by), "f"(v.z * by));
    *reinterpret_cast<uint2*>(P.out + (size_t)row * P.out_stride + (size_t)head * D + d) = r;
    if (P.lse && d == 0)
      P.lse[(size_t)row * P.H + head] = sum == 0.0f ? -INFINITY : __fmaf_rn(mx, kLn2, logf(sum));
  };
  // A piece's queries, as stored: row lane/4 of the tile (heads past the item's are zero), bf16
  // dims 8 (c + 4 i), e4m3 16 c + 64 (i / 2) + 8 (i % 2). They are asked for while the piece before
  // is merged, when its sums have left the registers.
  uint4 q_raw[kM][D / 32];
  auto load_q = [&](const PsCursor& p) {
    const int kvh = p.item / P.subs, sub = p.item - kvh * P.subs;
#pragma unroll
    for (int u = 0; u < kM; ++u) {
      const int h = sub * kHeads + 8 * u + hr;
      const uint4* q = reinterpret_cast<const uint4*>(P.q + (size_t)p.row * P.q_stride +
                                                      (size_t)(kvh * P.group + h) * D);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        q_raw[u][i] = make_uint4(0, 0, 0, 0);
        if (h < P.group) q_raw[u][i] = __ldg(q + (F8 ? 2 * c + 8 * (i / 2) + i % 2 : c + 4 * i));
      }
    }
  };
  load_q(piece);
  for (bool more_pieces = true; more_pieces;) {
    const PsRow keys = row_of(piece.row);
    const int row = piece.row;
    const int kvh = piece.item / P.subs, sub = piece.item - kvh * P.subs;
    const int head0 = kvh * P.group + sub * kHeads, heads = min(kHeads, P.group - sub * kHeads);
    const int lo = keys.low + piece.unit * unit;
    const int hi = (int)min((long long)keys.len, (long long)lo + (long long)piece.units * unit);
    const float vscale = F8 && P.v_scale ? P.v_scale[kvh] : 1.0f;

    // ---- Q's fragments
    uint32_t qa[kM][D / 16][2];
    float qk[kM];
#pragma unroll
    for (int u = 0; u < kM; ++u) {
      qk[u] = P.scale_log2;
      if (!F8) {
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) {
          qa[u][2 * i][0] = q_raw[u][i].x;
          qa[u][2 * i][1] = q_raw[u][i].y;
          qa[u][2 * i + 1][0] = q_raw[u][i].z;
          qa[u][2 * i + 1][1] = q_raw[u][i].w;
        }
      } else {
        float f[D / 4];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float2 p = unpack2<false>(word(q_raw[u][i], x));
            f[8 * i + 2 * x] = p.x;
            f[8 * i + 2 * x + 1] = p.y;
            top = fmaxf(top, fmaxf(fabsf(p.x), fabsf(p.y)));
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
            qa[u][i][x] = pack2<true>(f[4 * i + 2 * x] * down, f[4 * i + 2 * x + 1] * down);
        qk[u] *= up;
        if (P.k_scale) qk[u] *= P.k_scale[kvh];
      }
      // a factor above zero keeps the order of the scores (and -inf times it is -inf)
      if (qk[u] < 0.0f) {
        qk[u] = -qk[u];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) qa[u][i][x] ^= 0x80008000u;
      }
      qk[u] = fmaxf(qk[u], 1e-37f);
    }

    float o[kT][4];
#pragma unroll
    for (int i = 0; i < kT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] = 0.0f;
    float m[kM];
#pragma unroll
    for (int u = 0; u < kM; ++u) m[u] = -INFINITY;
    float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // sums of P, a product with a column of ones

    for (int base = lo + warp * S::kStep; base < hi; base += S::kUnit) {
      if (!wait_full(&full_s[warp][stage], phase, gave_up ? 0 : P.wait_ns,
                     P.skip_arrive == 2 && !gave_up && cta == 0 && tid == 5)) {
        gave_up = true;  // nothing more is issued: the stage's barrier may still be open
        more = false;
        if (lane == 0 && P.status) atomicOr(P.status, MC_KV_WAIT);
      }
      const uint32_t live = live_s[warp][stage] >> (S::kPart * c) & kAll;
      const uint8_t* k0 = ring + stage * S::kStage + k_at;
      const uint8_t* k1 = k0 + k_flip;
      const uint8_t* v0 = ring + stage * S::kStage + S::kHalf + v_at;
      const uint8_t* v1 = v0 + v_flip;
      // ---- scores; of key kPart c + 4 z + 2 j + x in t[u][z][2 j + x]
      float t[kM][kZ][4];
#pragma unroll
      for (int z = 0; z < kZ; ++z)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          auto a = [&](int u, int i, int x) { return u < kM ? qa[u % kM][i][x] : 0u; };
#pragma unroll
          for (int i = 0; i < kKLoads; ++i) {
            const uint4 w = *reinterpret_cast<const uint4*>(
                (i & 1 ? k1 : k0) + (4 * z + 2 * j) * S::kRow + 128 * (i >> 1));
            if (!F8) {
              mma16816<false>(s, a(0, 2 * i, 0), a(1, 2 * i, 0), a(0, 2 * i, 1), a(1, 2 * i, 1), w.x,
                              w.y);
              mma16816<false>(s, a(0, 2 * i + 1, 0), a(1, 2 * i + 1, 0), a(0, 2 * i + 1, 1),
                              a(1, 2 * i + 1, 1), w.z, w.w);
            } else {
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const int k = 4 * i + x;
                uint32_t b0, b1;
                e4m3x4_to_f16(word(w, x), b0, b1);
                mma16816<true>(s, a(0, k, 0), a(1, k, 0), a(0, k, 1), a(1, k, 1), b0, b1);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < kM; ++u) {
            t[u][z][2 * j] = s[2 * u];
            t[u][z][2 * j + 1] = s[2 * u + 1];
          }
        }
      // ---- running maxima
      if (live != kAll) {
#pragma unroll
        for (int i = 0; i < 4 * kZ; ++i)
          if (!(live >> i & 1u)) {
#pragma unroll
            for (int u = 0; u < kM; ++u) t[u][i / 4][i % 4] = -INFINITY;
          }
      }
      float m_use[kM], m_new[kM];
      bool grown = false;
#pragma unroll
      for (int u = 0; u < kM; ++u) {
        float top = fmaxf(fmaxf(t[u][0][0], t[u][0][1]), fmaxf(t[u][0][2], t[u][0][3]));
#pragma unroll
        for (int z = 1; z < kZ; ++z)
          top = fmaxf(top, fmaxf(fmaxf(t[u][z][0], t[u][z][1]), fmaxf(t[u][z][2], t[u][z][3])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // e4m3: see kUp; both roundings go up, so that no weight passes 2^kUp
        m_new[u] = fmaxf(m[u], F8 ? __fadd_ru(__fmul_ru(top, qk[u]), -kUp) : top * qk[u]);
        m_use[u] = m_new[u] == -INFINITY ? 0.0f : m_new[u];
        grown |= m_new[u] != m[u];
      }
      if (__any_sync(0xffffffffu, grown)) {
        float a[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) a[u] = ex2(m[u % kM] - m_use[u % kM]);
#pragma unroll
        for (int x = 0; x < 4; ++x) l4[x] *= a[x / 2];
#pragma unroll
        for (int i = 0; i < kT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i][x] *= a[x / 2];
#pragma unroll
        for (int u = 0; u < kM; ++u) m[u] = m_new[u];
      }
#pragma unroll
      for (int z = 0; z < kZ; ++z) {
        // P's high and low parts
        uint32_t high[kM][2], low[kM][2];
#pragma unroll
        for (int u = 0; u < kM; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float p0 = ex2(__fmaf_rn(t[u][z][2 * j], qk[u], -m_use[u]));
            const float p1 = ex2(__fmaf_rn(t[u][z][2 * j + 1], qk[u], -m_use[u]));
            high[u][j] = pack2<F8>(p0, p1);
            const float2 g = unpack2<F8>(high[u][j]);
            low[u][j] = pack2<F8>(p0 - g.x, p1 - g.y);
          }
        // 8 heads: the low parts are rows 8-15; 16 heads: a product of their own
        auto weigh = [&](float* sum, uint32_t b0, uint32_t b1) {
          if (kM == 1) {
            mma16816<F8>(sum, high[0][0], low[0][0], high[0][1], low[0][1], b0, b1);
          } else {
            mma16816<F8>(sum, high[0][0], high[kM - 1][0], high[0][1], high[kM - 1][1], b0, b1);
            mma16816<F8>(sum, low[0][0], low[kM - 1][0], low[0][1], low[kM - 1][1], b0, b1);
          }
        };
        uint32_t v[4][kVWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // an odd key's chunks lie in the other half of the line
          const uint8_t* vr = kHalfChunk ? (i & 1 ? v1 : v0) + 256 * z + 128 * (i >> 1)
                                         : (i & 1 ? v1 : v0) + (4 * z + i) * S::kRow;
          if (kHalfChunk) {
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
          if (live != kAll && !(live >> (4 * z + i) & 1u)) {
#pragma unroll
            for (int n = 0; n < kVWords; ++n) v[i][n] = 0u;
          }
        }
        constexpr uint32_t kOnes = F8 ? 0x3c003c00u : 0x3f803f80u;
        weigh(l4, kOnes, kOnes);
        // ---- o += P V
        if (!F8) {
#pragma unroll
          for (int i = 0; i < kT / 2; ++i) {
            weigh(o[2 * i], __byte_perm(v[0][i], v[1][i], 0x5410), __byte_perm(v[2][i], v[3][i], 0x5410));
            weigh(o[2 * i + 1], __byte_perm(v[0][i], v[1][i], 0x7632),
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
            for (int x = 0; x < 4; ++x) weigh(o[4 * i + x], b0[x], b1[x]);
          }
        }
      }
      if (++stage == S::kStages) {
        stage = 0;
        phase ^= 1;
      }
      __syncwarp();  // every lane has read the stage
      if (more) issue();
    }

    // ---- the warps' results of this piece
    if (kM == 1) {  // the low parts' rows
      l4[0] += l4[2];
#pragma unroll
      for (int i = 0; i < kT; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) o[i][x] += o[i][x + 2];
    }
    if (gave_up) l4[0] = l4[2] = __uint_as_float(0x7fc00000u);  // what did not arrive: NaN
    __syncthreads();  // the piece before is done with the shared arrays
#pragma unroll
    for (int u = 0; u < kM; ++u) {
      const int h = 8 * u + hr;
      if (c == 0) {
        m_s[warp][h] = m[u];
        l_s[warp][h] = l4[2 * u];
      }
#pragma unroll
      for (int i = 0; i < kT; i += 4)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          *reinterpret_cast<float4*>(o_s + (warp * kHeads + h) * S::kORow + v_dim<D, F8>(i, 2 * c + x)) =
              make_float4(o[i][2 * u + x], o[i + 1][2 * u + x], o[i + 2][2 * u + x],
                          o[i + 3][2 * u + x]);
    }
    const bool begins = piece.unit == 0, ends = piece.unit + piece.units == piece.n;
    const int n_units = piece.n, first_unit = u_end - piece.left - piece.unit;
    more_pieces = ps_next(piece, P.items, P.rows, units_of);
    if (more_pieces) load_q(piece);
    __syncthreads();
    float* part = P.parts + part_floats(D, kHeads) * (2 * (size_t)cta + (begins ? 1 : 0));
    for (int at = tid; at < heads * D / 4; at += S::kThreads) {
      const int h = 4 * at / D, d = 4 * at % D;
      float mx = m_s[0][h];
#pragma unroll
      for (int w = 1; w < S::kWarps; ++w) mx = fmaxf(mx, m_s[w][h]);
      const float use = mx == -INFINITY ? 0.0f : mx;
      float sum = 0.0f;
      float4 val = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < S::kWarps; ++w) {
        const float a = ex2(m_s[w][h] - use);
        const float4 u = *reinterpret_cast<const float4*>(o_s + (w * kHeads + h) * S::kORow + d);
        sum = __fmaf_rn(a, l_s[w][h], sum);
        val.x = __fmaf_rn(a, u.x, val.x);
        val.y = __fmaf_rn(a, u.y, val.y);
        val.z = __fmaf_rn(a, u.z, val.z);
        val.w = __fmaf_rn(a, u.w, val.w);
      }
      if (begins && ends) {
        finish(row, head0, vscale, at, mx, sum, val);
      } else {
        reinterpret_cast<float4*>(part)[at] = val;
        if (d == 0) {
          part[kHeads * D + h] = mx;
          part[kHeads * D + kHeads + h] = sum;
        }
      }
    }
    if (begins && ends) continue;
    // ---- the last of the item's CTAs joins the pieces in order
    const int first_cta = begins ? cta : ps_owner(first_unit, U, G);
    const int last_cta = ends ? cta : ps_owner(first_unit + n_units - 1, U, G);
    __syncthreads();
    if (tid == 0) {
      __threadfence();  // this CTA's part, written before the barrier
      const uint32_t done = atomicAdd(P.counters + first_cta, 1u);
      last_s = done == (uint32_t)(last_cta - first_cta);
      if (last_s) P.counters[first_cta] = 0;
      __threadfence();
    }
    __syncthreads();
    if (!last_s) continue;
    auto part_of = [&](int x) {
      return P.parts + part_floats(D, kHeads) * (2 * (size_t)x + (x == first_cta ? 1 : 0));
    };
    // Four elements a thread (or kQ times four), the pieces shared by `shares` threads for each, 12
    // loads of them in flight; the shares' results meet in o_s, which is free here.
    constexpr int kQ = (kHeads * D / 4 + S::kThreads - 1) / S::kThreads, kB = 12 / kQ;
    const int quads = heads * D / 4, shares = S::kThreads > quads ? S::kThreads / quads : 1;
    const int share = tid / quads, at0 = shares > 1 ? tid % quads : tid;
    float mx[kQ], sum[kQ];
    float4 val[kQ];
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      mx[q] = -INFINITY;
      sum[q] = 0.0f;
      val[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (share < shares || shares == 1)
      for (int x0 = first_cta + (shares > 1 ? share : 0); x0 <= last_cta; x0 += kB * shares) {
        float4 v[kQ][kB];
        float m8[kQ][kB], l8[kQ][kB];
#pragma unroll
        for (int k = 0; k < kB; ++k)
#pragma unroll
          for (int q = 0; q < kQ; ++q) {
            const int x = x0 + k * shares, at = at0 + q * S::kThreads;
            m8[q][k] = -INFINITY;
            l8[q][k] = 0.0f;
            v[q][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (x <= last_cta && at < quads) {
              const float* pp = part_of(x);
              v[q][k] = __ldcg(reinterpret_cast<const float4*>(pp) + at);
              m8[q][k] = __ldcg(pp + kHeads * D + 4 * at / D);
              l8[q][k] = __ldcg(pp + kHeads * D + kHeads + 4 * at / D);
            }
          }
#pragma unroll
        for (int q = 0; q < kQ; ++q) {
          float top = mx[q];
#pragma unroll
          for (int k = 0; k < kB; ++k) top = fmaxf(top, m8[q][k]);
          const float use = top == -INFINITY ? 0.0f : top, a0 = ex2(mx[q] - use);
          sum[q] *= a0;
          val[q] = make_float4(val[q].x * a0, val[q].y * a0, val[q].z * a0, val[q].w * a0);
          mx[q] = top;
#pragma unroll
          for (int k = 0; k < kB; ++k) {
            const float a = ex2(m8[q][k] - use);
            sum[q] = __fmaf_rn(a, l8[q][k], sum[q]);
            val[q].x = __fmaf_rn(a, v[q][k].x, val[q].x);
            val[q].y = __fmaf_rn(a, v[q][k].y, val[q].y);
            val[q].z = __fmaf_rn(a, v[q][k].z, val[q].z);
            val[q].w = __fmaf_rn(a, v[q][k].w, val[q].w);
          }
        }
      }
    if (shares == 1) {
#pragma unroll
      for (int q = 0; q < kQ; ++q)
        if (at0 + q * S::kThreads < quads) 
          finish(row, head0, vscale, at0 + q * S::kThreads, mx[q], sum[q], val[q]);
      continue;
    }
    float* stats = o_s + 4 * S::kThreads;
    if (share < shares) {
      reinterpret_cast<float4*>(o_s)[tid] = val[0];
      stats[2 * tid] = mx[0];
      stats[2 * tid + 1] = sum[0];
    }
    __syncthreads();
    if (tid < quads) {
      float top = -INFINITY, total = 0.0f;
      for (int k = 0; k < shares; ++k) top = fmaxf(top, stats[2 * (tid + k * quads)]);
      const float use = top == -INFINITY ? 0.0f : top;
      float4 o4 = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int k = 0; k < shares; ++k) {
        const int j = tid + k * quads;
        const float a = ex2(stats[2 * j] - use);
        const float4 u = reinterpret_cast<const float4*>(o_s)[j];
        total = __fmaf_rn(a, stats[2 * j + 1], total);
        o4.x = __fmaf_rn(a, u.x, o4.x);
        o4.y = __fmaf_rn(a, u.y, o4.y);
        o4.z = __fmaf_rn(a, u.z, o4.z);
        o4.w = __fmaf_rn(a, u.w, o4.w);
      }
      finish(row, head0, vscale, tid, top, total, o4);
    }
  }
  // copies still on their way end before the shared memory goes
  if (gave_up) mc_cp_async_wait_all();
}

template <int D, bool F8, int HEADS>
int launch_heads(mc_ctx* ctx, PaParams& P) {
  using S = Shape<D, F8, HEADS>;
  P.subs = (P.group + HEADS - 1) / HEADS;
  P.items = P.K * P.subs;
  const long long items = (long long)P.rows * P.items;
  P.small_unit = ps_small_unit(S::kUnit, items, P.capacity);
  if (P.small_unit == 0)
    return mc_fail(MC_EUNSUPPORTED, "paged_attention: %lld row and head groups", items);
  auto fn = paged_attention_kernel<D, F8, HEADS>;
  MC_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
  long long g = (long long)ctx->num_sms * S::kPerSm;
  const long long most = ((long long)P.capacity + S::kUnit - 1) / S::kUnit * items;
  if (g > most) g = most;
  if (g > kMaxCtas) g = kMaxCtas;
  MC_CUDA(mc_launch_pdl(fn, dim3((unsigned)g), dim3(S::kThreads), S::kSmem, ctx->stream, P));
  return mc_after_launch("paged_attention_kernel");
}

// Items of 8 heads, or of 16 where more share a KV head (see the rounding of P above).
template <int D, bool F8>
int launch_attention(mc_ctx* ctx, PaParams& P) {
  return P.group > 8 ? launch_heads<D, F8, 16>(ctx, P) : launch_heads<D, F8, 8>(ctx, P);
}

}  // namespace

extern "C" size_t mc_paged_attention_workspace_bytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128) return 0;
  return kCounterBytes + 2 * (size_t)kMaxCtas * part_floats(head_dim, 16) * sizeof(float);
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
  const long long capacity = (long long)table_width * block_size;
  PaParams P{q, q_stride, n_rows, n_heads, n_kv_heads, n_heads / n_kv_heads, 0, 0,
             k_cache, v_cache, num_blocks, block_size, (uint32_t)(block_stride / head_dim),
             ps_div_of(block_size), k_scale, v_scale, block_table, n_req, table_width,
             (int)(capacity < 0x7fff0000ll ? capacity : 0x7fff0000ll), 0, kv_lens, row_req, window,
             scale * kLog2e, out, out_stride, lse, static_cast<uint32_t*>(workspace),
             reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes), status,
             mc_wait_limit(ctx, 1000000000ull),
             ctx->test_flags & MC_TEST_SKIP_KV_ARRIVE   ? 1
             : ctx->test_flags & MC_TEST_LATE_KV_ARRIVE ? 2
                                                        : 0};
  const bool f8 = kv_dtype == MC_DTYPE_E4M3;
  if (head_dim == 64)
    return f8 ? launch_attention<64, true>(ctx, P) : launch_attention<64, false>(ctx, P);
  return f8 ? launch_attention<128, true>(ctx, P) : launch_attention<128, false>(ctx, P);
}
