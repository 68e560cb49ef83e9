// Causal grouped-query attention of decoded tokens over a cache held in 4 bits (packed_cache.cuh has the layout):
//   o = sum_j p_j v_j,  p = softmax_j(scale * q . k_j),  over the keys j of the request up to the token itself, the last `window` of them
// where a window is set.
//
// What bounds it is the cache's bytes, 9 D / 8 a position and KV head, as long as a position's codes become matrix operands in few
// instructions.  So the codes themselves are the operands, exactly, and steps and middles join on either side of the products:
//   a nibble c in a 16-bit half is the subnormal float16 c * 2^-24, one position higher 16 c * 2^-24: two elements by one AND, every
//   other pair by one shift more;
//   scores       s = scale * sum_g (step_g * (q . c)_g + (middle_g - 8 step_g) * (sum of q)_g), g the groups of 64 elements: keys are the rows
//                of the product (m16n8k16), the packed rows (tokens x query heads of the KV head) its columns;
//   values       o = sum_j (p_j step_j) (c_j - 8) + p_j middle_j: elements are the rows, keys the contraction; 8 times the sum of the very
//                weights comes from a product with a constant and goes off every 512 keys, so that the sums do not outgrow what they
//                stand for; the middles' sum on the CUDA cores in float32.  (The matrix unit lines products up by their operands' exponents, 2^-14 for any
//                subnormal, and cuts what lies 2^-24 or so below the largest: a sum of c * 2^-24 loses 2^-17 of 8 p step, less than a weight's rounding is worth at any
//                code but 8, one of 16 c * 2^-24 2^-21.  The 8 takes either form, so that the rows of each are cut alike.)
// Roundings: q, a power of two times itself that puts a row's largest element at 2^14 to 2^15, is a float16 (exactly, from bfloat16 also, but for what is
// 2^-30 below the largest); p step, times a power of two that follows the largest one seen by the row in the group, is rounded to float16: a weight's half
// step of 2^-12, and the result's own.  All sums are float32: an element's weighted sum, values times keys times 2^SLACK at most, has to stay in it.
// (A power of two of the warp's own instead of each row's and group's took the bits of values that are 2^26 times smaller than what another row, or the other half of
// a head, looks at; B200, us, it / each its own: 64 x 8,192 keys 134.8 / 134.0, one of 700 9.6 / 9.8, 17 x up to 6,000, 4 tokens each, 42 / 44, 8 x 8,192 with 16
// heads a KV head 25.4 / 26.9.)
//
// The work is handed out on the device, so that the launch does not depend on the lengths and a captured one serves any.  A (request, KV head,
// rows of 8 NT) is a pair.  Few pairs (OWN CTAs or more for each): each gets a number of CTAs of its own by its length, one part a CTA, of NB units at
// least (a step takes as long with one), as a part costs some 4 us beside its keys.  Many: they form one line, a pair as long as its units of 64 keys and EXTRA for
// that cost, and CTA c of P takes the stretch [c L / P, (c + 1) L / P); pairs of up to WHOLE units (and of no more than a stretch) are not cut but belong
// to the CTA in whose stretch they begin.  B200, bfloat16, us (D 128, 8 KV heads, where nothing else is said):
//   OWN 2 / 3: 17 requests of up to 6,000 keys, 4 tokens each 46 / 44; a line always: 17 in a window of 2,000, D 64, 14.9 -> 16.0; parts of one unit: 100 keys 7.6 -> 9.1
//   EXTRA 0 / 6 / 12: 40 requests of 30 to 900 keys, 32 KV heads 113 / 47 / 50, 64 x 8,192 keys 139 / 135 / 134, 40 x 30 to 900 keys 33 / 21 / 20
//   WHOLE 0 / 16 / 64: 64 x 200 keys 21.5 / 18.3 / 18.2, 40 x 465 keys, 32 KV heads 49 / 38 / 38, 64 x 400 to 2,000 keys 36.8 / 36.9 / 39.4
// A CTA's four warps take every fourth block of 16 positions; a block is one bulk copy into the warp's own ring of stages, and no
// warp waits for another until its part is done; the first copies of the next part are on their way by then.  Of the CTAs that share a (request, head) the one that comes last adds up the parts, in a fixed order.
//
// Measured (B200, bfloat16, D 128, 32 heads on 8 KV heads, in a CUDA graph): 64 requests of 8,192 keys 134 us, 4.5 TB/s of cache where a copy runs at 6.6; one of
// 131,000 keys 43 us, 3.5 TB/s; 64 of 200 keys 18.2 us; one of 700 keys 9.8 us.  What bounds the long ones is the chain of instructions from a block's codes to its
// sums, which the 11 warps that an SM's registers hold do not hide: 55 % of the issue slots, 54 % of the ALU, 27 % of the matrix pipe, 52 % of the
// DRAM are busy, and with the copies alone the same kernel takes 107 us.  Two CTAs an SM take 147 us; longer rings or steps of four blocks, for
// which the third CTA goes, were no faster.
#include "packed_cache.cuh"
#include "ptx_sm100.cuh"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int WARPS = 4;
constexpr int TILE = WARPS * PACKED_POS;     // keys of a unit
constexpr int NB = 2;                        // blocks of a step: one running maximum for 32 keys
constexpr float SLACK = 6.f;                 // a weight is at most 2^SLACK times that of the maximum in use
constexpr float FAR = 0x1p24f;               // scores of which float32 holds whole numbers at best
constexpr int HEAD = 10;                     // a row's largest p step, when v_up is set by it, comes to 2^(HEAD - 1) to 2^HEAD: 2^6 of room
constexpr float BEHIND = 6.f;                // the maximum may rise by so much until v_up follows
constexpr int V_UP_MOST = 115;               // (its exponent: bfloat16's smallest normal steps come to 2^-11 with it)
constexpr int SETTLE = 16;                   // steps after which the sums of codes are centred
constexpr int HALVES = 2;                    // steps in a warp's ring: one is read while the next arrives
static_assert(32 % NB == 0, "the blocks of a step lie in one window of 32 blocks, one a lane");
constexpr int OWN = 3;                       // pairs get CTAs of their own where there are this many CTAs for each
constexpr int EXTRA = 6;                     // what a part costs beside its keys, in units
constexpr int WHOLE = 16;                    // units up to which a pair is not cut
constexpr int PART_ROWS = 16;                // rows of a partial's slot

struct PackedParams {
  const void* q;
  void* out;
  const uint8_t* plane;
  const int* block_table;
  const int* q_start;
  const int* pos0;
  float* part_o;        // [2 P][PART_ROWS][D]
  float* part_ml;       // [2 P][PART_ROWS][2]
  int* counters;        // [requests * Hkv * 2], zeros before and after: the parts of a (request, head, row tile) that are there
  int* err;
  long long page_stride;
  int ldq, ldo, n_pages, page_size, table_width, table_keys, Hq, Hkv, G, window, n_reqs;
  float scale_log2;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// c += a b, or c = a b for the first product of a sum.
__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1, bool first = false) {
  if (first)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8(unsigned v) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ float2 pair_values(unsigned v);
template <> __device__ __forceinline__ float2 pair_values<__nv_bfloat16>(unsigned v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
template <> __device__ __forceinline__ float2 pair_values<__half>(unsigned v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }

// Two results, rounded.  The rounding of a step may carry a group's outermost levels beyond the type, which what they stand for is not: the type's largest number then,
// as for an infinity (a sum that has left float32); a NaN stays one.
template <typename T> __device__ __forceinline__ unsigned pack2_within(float lo, float hi);
template <> __device__ __forceinline__ unsigned pack2_within<__nv_bfloat16>(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ unsigned pack2_within<__half>(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int N>
__device__ __forceinline__ void load_words(unsigned (&w)[N], const uint8_t* p) {
  if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x;
    w[N - 1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const unsigned*>(p);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {      // 2 ulp; below 2^-126: 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Waits for a copy, about a second at most (a moment once one has failed to come).
__device__ __forceinline__ bool arrived(uint32_t bar, uint32_t parity, bool failed) {
  if (sm100::mbar_try_wait(bar, parity)) return true;
  const long long begin = clock64(), limit = failed ? 1000000 : sm100::WAIT_LIMIT_CYCLES;
  while (clock64() - begin <= limit)
    if (sm100::mbar_try_wait(bar, parity)) return true;
  return false;
}

// CTAs that an SM holds, as the registers of the accumulators allow.
template <int D, int NT>
constexpr int RESIDENT = NT == 1 ? 3 : D == 64 ? 3 : 2;
constexpr int MAX_RESIDENT = 4;

// A request's part of the line.
struct Span {
  int lo, tiles, row_tiles;      // first key (a block's first), tiles of TILE keys (none: not a request of few rows, or a bad one, which has rows), tiles of rows
};
template <int NT>
__device__ __forceinline__ Span span_of(const PackedParams& p, int r) {
  const int n = p.q_start[r + 1] - p.q_start[r], rows = n * p.G;
  if (rows <= 0 || rows > PACKED_FEW_ROWS) return Span{0, 0, 0};
  const int pos = p.pos0[r];
  if ((unsigned)pos > (unsigned)(p.table_keys - n)) return Span{0, 0, rows};      // keys that no page of the table could hold (n <= 16 <= table_keys)
  const int lo = (p.window > 0 ? max(0, pos - p.window + 1) : 0) / PACKED_POS * PACKED_POS;
  return Span{lo, (pos + n - lo + TILE - 1) / TILE, (rows + 8 * NT - 1) / (8 * NT)};
}

// Where the parts of a pair lie: n CTAs from `cta` on; the first one's is in the odd slot of its two (the pair ends beyond that CTA's stretch), the others'
// in the even slots of theirs.  n = 1: not cut.
struct Parts {
  int cta, n;
  __device__ __forceinline__ int slot(int i) const { return 2 * (cta + i) + (i == 0); }
};

template <typename T>
__device__ __forceinline__ void write_row4(const PackedParams& p, int token, int head, int D, int d, float4 acc, float L) {
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  uint2 r;
  r.x = pack2_within<T>(acc.x * inv, acc.y * inv);
  r.y = pack2_within<T>(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>((T*)p.out + (size_t)token * p.ldo + (size_t)head * D + d) = r;
}

// How the work is shared out: the line's length, units and pairs in all, CTAs, the CTA's own stretch of the line (or its own part, where pairs have
// CTAs of their own).
struct Way {
  long long L, U, P, N, first, last;
  int whole;              // pairs of up to so many units are not cut
  bool own;
};

// A CTA's part of a pair: blocks [q0, q1) of 16 positions from key_lo on.
struct Item {
  int r, kvh, rt, key_lo, q0, q1;
  Parts parts;
};

// A warp's way through the blocks of an item: b0, b0 + WARPS, ..., n_blocks of them.  Where the next 32 of them lie is kept one a lane, which also asks
// for its copy when its step's turn comes.
template <int D>
struct Flow {
  using B = PackedBlock<D>;
  const int* bt;
  const uint8_t* head;
  const uint8_t* my_src;
  int key_lo, b0, n_blocks;

  __device__ __forceinline__ void find(const PackedParams& p, int i, int lane) {      // blocks i .. i + 31 of the warp
    const int k = i + lane;
    if (k < n_blocks) {
      const int key = key_lo + (b0 + k * WARPS) * PACKED_POS, lp = key / p.page_size;
      int page = lp < p.table_width ? bt[lp] : -1;
      if (page < 0 || page >= p.n_pages) {      // the flag fails the step; the request's rows are nobody's then, and page 0 will do
        atomicExch(p.err, 5);
        page = 0;
      }
      my_src = head + (size_t)page * p.page_stride + (size_t)((key - lp * p.page_size) / PACKED_POS) * B::BYTES;
    }
  }
  // the copies of step j (blocks NB j .. NB j + NB - 1, those that there are), the warp's step number `turn`
  __device__ __forceinline__ void request(const PackedParams& p, int j, uint32_t turn, uint8_t* ring, uint32_t bars, int lane) {
    if ((NB * j & 31) == 0) find(p, NB * j, lane);
    const uint32_t half = turn % HALVES, bar = bars + 8 * half;
    const int b = lane - (NB * j & 31), n = min(NB, n_blocks - NB * j);
    if (b == 0) sm100::mbar_expect_tx(bar, n * B::BYTES);
    if (b >= 0 && b < n) bulk_load(sm100::smem_u32(ring + (half * NB + b) * B::BYTES), my_src, B::BYTES, bar);
  }
  __device__ __forceinline__ int steps() const { return (n_blocks + NB - 1) / NB; }
  __device__ __forceinline__ void begin(const PackedParams& p, const Item& it, uint32_t turn, uint8_t* ring, uint32_t bars) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    bt = p.block_table + (size_t)it.r * p.table_width;
    head = p.plane + (size_t)it.kvh * (p.page_size / PACKED_POS) * B::BYTES;
    my_src = head;
    key_lo = it.key_lo;
    b0 = it.q0 + warp;
    n_blocks = b0 < it.q1 ? (it.q1 - b0 + WARPS - 1) / WARPS : 0;
    for (int j = 0; j < min(HALVES, steps()); ++j) request(p, j, turn + j, ring, bars, lane);
  }
};

// One item, whose first copies are on their way; next() sends the next item's.
template <typename T, int D, int NT, typename Next>
__device__ __forceinline__ void packed_item(const PackedParams& p, const Item it, Flow<D>& flow, uint8_t* ring, uint32_t bars, uint32_t& turn, float* merge, bool& failed,
                                            Next next) {
  using B = PackedBlock<D>;
  constexpr int GN = B::GROUPS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  const int r = it.r, kvh = it.kvh, rt = it.rt;
  const Parts parts = it.parts;
  const int qs = p.q_start[r], n_rows = (p.q_start[r + 1] - qs) * p.G, pos0 = p.pos0[r];
  const int row0 = rt * 8 * NT;
  const int hi = pos0 + p.q_start[r + 1] - qs;                       // one past the last key
  const int n_blocks = flow.n_blocks, n_steps = flow.steps();

  // ---- the rows' queries as float16 operands, their sums per group and their scale
  unsigned qf[NT][GN][4][2];
  float q_sum[NT][GN][2], f_row[NT][2];
  int e_row[NT], e_least = 126;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int row = row0 + nt * 8 + gid;
    float x[GN][16], big = 0.f;
#pragma unroll
    for (int g = 0; g < GN; ++g) {
      uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (row < n_rows) {
        const uint4* src = reinterpret_cast<const uint4*>((const T*)p.q + (size_t)(qs + row / p.G) * p.ldq + (size_t)(kvh * p.G + row % p.G) * D + g * PACKED_GROUP + tig * 16);
        raw[0] = src[0];
        raw[1] = src[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = pair_values<T>(reinterpret_cast<const unsigned*>(raw)[i]);
        x[g][2 * i] = v.x;
        x[g][2 * i + 1] = v.y;
        big = fmaxf(big, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // 2^e brings the largest element to [2^14, 2^15); bfloat16's largest numbers to 65,280 at most, which a float16 still holds; its smallest to
    // what a float's exponents allow
    const int e = max(-112, min(126, 14 + 127 - (int)(__float_as_uint(big) >> 23)));
    e_least = min(e_least, e);
    e_row[nt] = e;
    const float up = copysignf(__uint_as_float((unsigned)(127 + e) << 23), p.scale_log2);      // (f_row is not negative: it orders the scores)
    float sum[GN];
#pragma unroll
    for (int g = 0; g < GN; ++g) {
      sum[g] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[g][i] = __half2float(__float2half_rn(x[g][i] * up));
        sum[g] += x[g][i];
      }
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
      sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {      // step 2 j + h of the contraction: nibbles 2 h and 2 h + 4, then 2 h + 1 and 2 h + 5 (16 times as large)
          qf[nt][g][2 * j + h][0] = pack2<__half>(x[g][8 * j + 2 * h], x[g][8 * j + 2 * h + 4]);
          qf[nt][g][2 * j + h][1] = pack2<__half>(x[g][8 * j + 2 * h + 1] * 0.0625f, x[g][8 * j + 2 * h + 5] * 0.0625f);
        }
    }
    // the scores' columns: this thread meets rows 2 tig and 2 tig + 1
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int g = 0; g < GN; ++g) q_sum[nt][g][c] = __shfl_sync(0xffffffffu, sum[g], (2 * tig + c) * 4) * 0x1p-24f;
  }
  // A score is f_row, 2^24 scale 2^-e, times a sum that the keys' steps and middles make.  Under queries of 2^90 and more the one would leave float32 and the other
  // its normal numbers: 2^shift moves from the factor to the keys then (whose own elements are far below 2^90 where the scores are to be finite).
  constexpr bool WIDE_Q = std::is_same<T, __nv_bfloat16>::value;
  const int shift = WIDE_Q ? max(0, -76 - __reduce_min_sync(0xffffffffu, e_least)) : 0;
  const float k_up = __uint_as_float((unsigned)(127 + shift) << 23);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float f = fabsf(p.scale_log2) * __uint_as_float((unsigned)(127 + 24 - shift) << 23) * __uint_as_float((unsigned)(127 - e_row[nt]) << 23);
#pragma unroll
    for (int c = 0; c < 2; ++c) f_row[nt][c] = __shfl_sync(0xffffffffu, f, (2 * tig + c) * 4);
  }
  // keys that every row sees: from the last row's window on, up to the first row's position
  const int all_hi = pos0 + row0 / p.G, all_lo = p.window > 0 ? max(0, pos0 + (min(n_rows, row0 + 8 * NT) - 1) / p.G - p.window + 1) : 0;

  float m_run[NT][2], l_run[NT][2], mid_acc[NT][GN][2], o[NT][GN][4][4], eights[NT][GN][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m_run[nt][c] = -INFINITY;
      l_run[nt][c] = 0.f;
#pragma unroll
      for (int g = 0; g < GN; ++g) {
        mid_acc[nt][g][c] = eights[nt][g][c] = eights[nt][g][2 + c] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[nt][g][j][c] = o[nt][g][j][2 + c] = 0.f;
      }
    }
  // what p step is multiplied by before it becomes a float16 operand: of each row and group its own, so that no row, and no half of a head, loses bits to another
  float v_up[NT][GN][2], m_up[NT][2];      // (m_up: the maximum that v_up goes by)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int g = 0; g < GN; ++g) v_up[nt][g][0] = v_up[nt][g][1] = __uint_as_float((unsigned)(127 + V_UP_MOST) << 23);

  // whole blocks, by their number in the warp: [k_lo, k_hi) hide no key from any row
  const int base = flow.key_lo + flow.b0 * PACKED_POS;
  const int k_lo = all_lo > base ? (all_lo - base + TILE - 1) / TILE : 0;
  int k_hi = shift == 0 && all_hi - PACKED_POS + 1 >= base ? (all_hi - PACKED_POS + 1 - base) / TILE + 1 : 0;

  // v_up and the sums that hold it, times 2^by
  auto scale_up = [&](int nt, int g, int c, int by) {
    const float ratio = by < -126 ? 0.f : __uint_as_float((unsigned)(127 + min(by, 127)) << 23);      // (by 2^127 and more: what float32's weights had shrunk to nothing)
    v_up[nt][g][c] = __uint_as_float(__float_as_uint(v_up[nt][g][c]) + ((unsigned)by << 23));
    eights[nt][g][c] *= ratio;
    eights[nt][g][2 + c] *= ratio;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[nt][g][j][c] *= ratio;
      o[nt][g][j][2 + c] *= ratio;
    }
  };
  // (m_run: the maximum in use, a score times f_row.  Its own rounding is a part of a fused exponent, which from scores of FAR on is no longer small: the steps
  // that follow take the masked form, whose exponents are not fused.)
  // The step's blocks, the first at key0.  MASKED: some key of theirs is hidden from some row or lies behind the last key, or queries or scores are
  // so large that they want its ways.
  auto step_of = [&](auto masked, const uint8_t* const first, const int key0, const int n) {
    constexpr bool MASKED = decltype(masked)::value;
    // ---- scores, still to be multiplied by f_row
    float s[NB][NT][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float part[NT][GN][4];
      unsigned wu[GN][2], wv[GN][2];       // keys gid and gid + 8
#pragma unroll
      for (int g = 0; g < GN; ++g) {
        load_words<2>(wu[g], first + b * B::BYTES + gid * B::ROW + g * 32 + tig * 8);
        load_words<2>(wv[g], first + b * B::BYTES + (gid + 8) * B::ROW + g * 32 + tig * 8);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int g = 0; g < GN; ++g) {
            const unsigned u = wu[g][j] >> (8 * h), v = wv[g][j] >> (8 * h);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(part[nt][g], u & 0x000F000Fu, v & 0x000F000Fu, u & 0x00F000F0u, v & 0x00F000F0u, qf[nt][g][2 * j + h][0], qf[nt][g][2 * j + h][1], j + h == 0);
          }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        unsigned pairs[GN];
        load_words<GN>(pairs, first + b * B::BYTES + B::K_PAIRS + (gid + 8 * k) * GN * 4);
#pragma unroll
        for (int g = 0; g < GN; ++g) {
          float2 v = pair_values<T>(pairs[g]);
          if (MASKED && WIDE_Q) v.x *= k_up, v.y *= k_up;
          const float mid = fmaf(-8.f, v.x, v.y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float& t = s[b][nt][2 * k + c];
              t = fmaf(v.x, part[nt][g][2 * k + c], g == 0 ? mid * q_sum[nt][g][c] : fmaf(mid, q_sum[nt][g][c], t));
            }
        }
      }
      if (MASKED) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + b * TILE + gid + 8 * (e >> 1), row = row0 + nt * 8 + 2 * tig + (e & 1);
            const int at = pos0 + row / p.G;
            if (b >= n || key > at || (p.window > 0 && key <= at - p.window) || key >= hi) s[b][nt][e] = -INFINITY;
          }
      }
    }
    // ---- the values' steps and middles
    float step[NB][GN][2], mid[NB][GN][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        unsigned pairs[GN];
        load_words<GN>(pairs, first + b * B::BYTES + B::V_PAIRS + (gid + 8 * k) * GN * 4);
#pragma unroll
        for (int g = 0; g < GN; ++g) {
          float2 v = pair_values<T>(pairs[g]);
          if (MASKED && (b >= n || key0 + b * TILE + gid + 8 * k >= hi)) v = make_float2(0.f, 0.f);      // (what lies behind the last key may be a NaN)
          step[b][g][k] = v.x;
          mid[b][g][k] = v.y;
        }
      }
    // ---- exponents against the maximum in use, which moves only when a score leaves it 2^SLACK behind: a vote in its place otherwise
    float x[NB][NT][4], far = -INFINITY;
    if (!MASKED) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            x[b][nt][e] = fmaf(s[b][nt][e], f_row[nt][e & 1], -m_run[nt][e & 1]);
            far = fmaxf(far, x[b][nt][e]);
          }
    }
    if (MASKED || __any_sync(0xffffffffu, far > SLACK)) {
      bool large = false, behind = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(s[0][nt][c], s[0][nt][2 + c]);
#pragma unroll
          for (int b = 1; b < NB; ++b) mx = fmaxf(mx, fmaxf(s[b][nt][c], s[b][nt][2 + c]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_new = fmaxf(m_run[nt][c], mx == -INFINITY ? mx : mx * f_row[nt][c]);
          // (nothing seen so far: the sums are zeros)
          const float corr = m_run[nt][c] == -INFINITY ? 0.f : exp2_fast(m_run[nt][c] - m_new);
          if (m_run[nt][c] == -INFINITY) m_up[nt][c] = m_new;
          m_run[nt][c] = m_new;
          behind |= m_new - m_up[nt][c] > BEHIND;
          large |= fabsf(m_new) >= FAR && m_new != -INFINITY;
          l_run[nt][c] *= corr;
#pragma unroll
          for (int g = 0; g < GN; ++g) {
            mid_acc[nt][g][c] *= corr;
            eights[nt][g][c] *= corr;
            eights[nt][g][2 + c] *= corr;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[nt][g][j][c] *= corr;
              o[nt][g][j][2 + c] *= corr;
            }
          }
        }
      if (__any_sync(0xffffffffu, large)) k_hi = 0;
      // The largest product so far has shrunk with the sums, by 2^BEHIND and more: v_up and the sums rise by what it was, so that what is left of it is where it was, and
      // products of smaller steps keep their bits.
      if (__any_sync(0xffffffffu, behind)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int most = (int)fminf(m_run[nt][c] - m_up[nt][c], 300.f);
            m_up[nt][c] = m_run[nt][c];
#pragma unroll
            for (int g = 0; g < GN; ++g) scale_up(nt, g, c, min(most, V_UP_MOST + 127 - (int)(__float_as_uint(v_up[nt][g][c]) >> 23)));
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < NB; ++b)      // (the product rounded as the maximum was: its own exponent is 0 whatever its size)
            x[b][nt][e] = MASKED && s[b][nt][e] == -INFINITY ? -INFINITY : __fsub_rn(__fmul_rn(s[b][nt][e], f_row[nt][e & 1]), m_run[nt][e & 1]);
    }
    // ---- weights; times a step and v_up they are float16 operands
    float w[NB][NT][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[b][nt][e] = exp2_fast(x[b][nt][e]);
          l_run[nt][e & 1] += w[b][nt][e];
        }
    // Where a product has left float16: v_up of each row and group whose largest one in the step is beyond 2^HEAD goes down to where it is 2^(HEAD - 1) to 2^HEAD.
    auto lower = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < GN; ++g) {
          unsigned both = 0;           // the exponents of two columns' largest products
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) top = fmaxf(top, fmaxf(w[b][nt][c] * step[b][g][0], w[b][nt][2 + c] * step[b][g][1]));      // (hidden keys' NaN are passed over)
            both |= __float_as_uint(top) >> 23 << (16 * c);
          }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // top < 2^(top - 126); a product beyond float32: a weight of 2^SLACK takes it to 2^132 at most
            const int top = both >> (16 * c) & 255, now = (int)(__float_as_uint(v_up[nt][g][c]) >> 23) - 127;
            scale_up(nt, g, c, min(0, HEAD - (top == 255 ? 132 : top - 126) - now));
          }
        }
    };
    unsigned pf[NB][NT][GN][2];
    auto operands = [&]() {      // returns whether one is beyond a float16
      __half2 most = __float2half2_rn(0.f);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int g = 0; g < GN; ++g)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              // (the weight first: what a row looks away from is 0 whatever its step is)
              float y0 = w[b][nt][2 * k] * v_up[nt][g][0] * step[b][g][k], y1 = w[b][nt][2 * k + 1] * v_up[nt][g][1] * step[b][g][k];
              if (MASKED) {            // a key that a row does not see counts for nothing, whatever it holds
                if (w[b][nt][2 * k] == 0.f) y0 = 0.f;
                if (w[b][nt][2 * k + 1] == 0.f) y1 = 0.f;
              }
              pf[b][nt][g][k] = pack2<__half>(y0, y1);
              most = __hmax2(most, *reinterpret_cast<__half2*>(&pf[b][nt][g][k]));
            }
      const unsigned bits = *reinterpret_cast<unsigned*>(&most);
      return (bits & 0xffffu) >= 0x7c00u || bits >= 0x7c000000u;
    };
    if (__any_sync(0xffffffffu, operands())) {
      lower();
      operands();
    }
    // ---- values
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int g = 0; g < GN; ++g) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (!MASKED || w[b][nt][2 * k] != 0.f) mid_acc[nt][g][0] = fmaf(w[b][nt][2 * k], mid[b][g][k], mid_acc[nt][g][0]);
            if (!MASKED || w[b][nt][2 * k + 1] != 0.f) mid_acc[nt][g][1] = fmaf(w[b][nt][2 * k + 1], mid[b][g][k], mid_acc[nt][g][1]);
            pf[b][nt][g][k] = transpose8(pf[b][nt][g][k]);
          }
          mma_f16(eights[nt][g], 0x00080008u, 0x00800080u, 0x00080008u, 0x00800080u, pf[b][nt][g][0], pf[b][nt][g][1]);
        }
      }
      // keys of the contraction: index 2 tig + i of the first half is row tig * 2 + i of the block, of the second half 8 more
#pragma unroll
      for (int g = 0; g < GN; ++g) {
        unsigned w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = *reinterpret_cast<const unsigned*>(first + b * B::BYTES + B::V_CODES + (2 * tig + (k & 1) + 8 * (k >> 1)) * B::ROW + g * 32 + gid * 4);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          unsigned x = __byte_perm(w[0], w[1], half ? 0x7632 : 0x5410), y = __byte_perm(w[2], w[3], half ? 0x7632 : 0x5410);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_f16(o[nt][g][2 * half + h], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pf[b][nt][g][0], pf[b][nt][g][1]);
            x >>= 8;
            y >>= 8;
          }
        }
      }
    }
  };

  // The 8 of (c - 8) comes off the sums now and then: they grow with the keys otherwise, and what they stand for does not.
  auto settle = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int g = 0; g < GN; ++g)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            o[nt][g][j][c] -= eights[nt][g][c];
            o[nt][g][j][2 + c] -= eights[nt][g][2 + c];
          }
          eights[nt][g][c] = eights[nt][g][2 + c] = 0.f;
        }
  };
  for (int j = 0; j < n_steps; ++j) {
    const uint32_t half = (turn + j) % HALVES;
    failed |= !arrived(bars + 8 * half, (turn + j) / HALVES & 1, failed);
    const uint8_t* first = ring + half * NB * B::BYTES;
    if (NB * j >= k_lo && NB * j + NB <= min(k_hi, n_blocks)) step_of(std::false_type{}, first, 0, NB);
    else step_of(std::true_type{}, first, base + NB * j * TILE, n_blocks - NB * j);
    if (j % SETTLE == SETTLE - 1) settle();
    __syncwarp();                      // the half is free
    if (j + HALVES < n_steps) flow.request(p, j + HALVES, turn + j + HALVES, ring, bars, lane);
  }
  settle();
  turn += n_steps;
  if (failed) atomicExch(p.err, 29);
  next();

  // ---- the warps' parts meet, eight rows at a time
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l_run[nt][c] += __shfl_xor_sync(0xffffffffu, l_run[nt][c], d);
#pragma unroll
        for (int g = 0; g < GN; ++g) mid_acc[nt][g][c] += __shfl_xor_sync(0xffffffffu, mid_acc[nt][g][c], d);
      }
    }
    float* ml = merge + WARPS * 8 * D;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 2 * tig + c;
      if (gid == 0) {
        ml[(warp * 8 + row) * 2] = m_run[nt][c];
        ml[(warp * 8 + row) * 2 + 1] = l_run[nt][c];
      }
#pragma unroll
      for (int g = 0; g < GN; ++g)
#pragma unroll
        for (int j = 0; j < 4; ++j) {      // tile j of the group: elements 8 gid + 2 j and, 16 times as large, 8 gid + 2 j + 1
          const float down = __uint_as_float((254u << 23) - __float_as_uint(v_up[nt][g][c]));      // its reciprocal
          float2 v = make_float2(fmaf(o[nt][g][j][c] * 0x1p24f, down, mid_acc[nt][g][c]), fmaf(o[nt][g][j][2 + c] * 0x1p20f, down, mid_acc[nt][g][c]));
          *reinterpret_cast<float2*>(merge + (warp * 8 + row) * D + g * PACKED_GROUP + 8 * gid + 2 * j) = v;
        }
    }
    __syncthreads();
    for (int idx = tid; idx < 8 * (D / 4); idx += WARPS * 32) {
      const int rr = idx / (D / 4), d = idx % (D / 4) * 4, row = row0 + nt * 8 + rr;
      if (row >= n_rows) continue;
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) M = fmaxf(M, ml[(w * 8 + rr) * 2]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float mw = ml[(w * 8 + rr) * 2], f = mw == -INFINITY ? 0.f : exp2f(mw - M);
        const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + rr) * D + d);
        L += ml[(w * 8 + rr) * 2 + 1] * f;
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
      }
      if (parts.n == 1) {
        write_row4<T>(p, qs + row / p.G, kvh * p.G + row % p.G, D, d, acc, L);
      } else {
        const size_t at = (size_t)parts.slot((int)blockIdx.x - parts.cta) * PART_ROWS + nt * 8 + rr;
        __stcg(reinterpret_cast<float4*>(p.part_o + at * D + d), acc);
        if (d == 0) __stcg(reinterpret_cast<float2*>(p.part_ml + at * 2), make_float2(M, L));
      }
    }
  }
  if (parts.n == 1) return;
  // ---- the last CTA to come adds the parts up
  __shared__ int s_last;
  __syncthreads();
  if (tid == 0) {
    int* count = p.counters + ((size_t)r * p.Hkv + kvh) * 2 + rt;
    int before;                        // (the block's stores come before it by the barrier, what the others stored before theirs by theirs)
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(count) : "memory");
    s_last = before == parts.n - 1;
    if (s_last) *count = 0;
  }
  __syncthreads();
  if (!s_last) return;
  // CHUNK parts at a time: a warp a row forms the parts' factors, then a thread adds four elements of a row over the parts, all loads in flight
  constexpr int CHUNK = 64, ITEMS = 8 * NT * (D / 4) / (WARPS * 32), GROUP = 16;
  const int rows = min(8 * NT, n_rows - row0);
  float* factor = merge;               // [8 NT][CHUNK]
  float* state = merge + 8 * NT * CHUNK;      // [8 NT][3]: maximum, sum, what becomes of the sums so far
  float4 acc[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto load_parts = [&](float4 (&v)[GROUP], int i0, int n, int rr, int d) {      // parts i0 .., of which the last is n - 1
#pragma unroll
    for (int i = 0; i < GROUP; ++i) v[i] = __ldcg(reinterpret_cast<const float4*>(p.part_o + ((size_t)parts.slot(min(i0 + i, n - 1)) * PART_ROWS + rr) * D + d));
  };
  for (int first = 0; first < parts.n; first += CHUNK) {
    const int n = min(CHUNK, parts.n - first);
    float4 ahead[GROUP];               // (the first loads go out before the factors are known)
    load_parts(ahead, first, first + n, min(tid / (D / 4), rows - 1), tid % (D / 4) * 4);
    for (int rr = warp; rr < rows; rr += WARPS) {
      float2 ml[CHUNK / 32];
      float m_run = first ? state[rr * 3] : -INFINITY, m_new = m_run;
#pragma unroll
      for (int k = 0; k < CHUNK / 32; ++k) {
        const int i = lane + 32 * k;
        ml[k] = i < n ? __ldcg(reinterpret_cast<const float2*>(p.part_ml + ((size_t)parts.slot(first + i) * PART_ROWS + rr) * 2)) : make_float2(-INFINITY, 0.f);
        m_new = fmaxf(m_new, ml[k].x);
      }
      m_new = warp_max(m_new);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < CHUNK / 32; ++k) {
        const float f = ml[k].x == -INFINITY && ml[k].y == 0.f ? 0.f : exp2f(ml[k].x - m_new);      // (a part of which the row sees no key: zeros)
        sum += ml[k].y * f;
        factor[rr * CHUNK + lane + 32 * k] = f;
      }
      sum = warp_sum(sum);
      if (lane == 0) {
        const float keep = m_run == -INFINITY ? 0.f : exp2f(m_run - m_new);
        state[rr * 3 + 1] = first ? state[rr * 3 + 1] * keep + sum : sum;
        state[rr * 3 + 2] = keep;
        state[rr * 3] = m_new;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int idx = tid + k * WARPS * 32, rr = idx / (D / 4), d = idx % (D / 4) * 4;
      if (rr >= rows) continue;
      const float keep = state[rr * 3 + 2];
      acc[k].x *= keep; acc[k].y *= keep; acc[k].z *= keep; acc[k].w *= keep;
      for (int i0 = 0; i0 < n; i0 += GROUP) {
        float4 v[GROUP];
        if (k == 0 && i0 == 0) {
#pragma unroll
          for (int i = 0; i < GROUP; ++i) v[i] = ahead[i];
        } else {
          load_parts(v, first + i0, first + n, rr, d);
        }
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
          const float f = factor[rr * CHUNK + i0 + i];      // (0 behind the last part)
          acc[k].x += v[i].x * f; acc[k].y += v[i].y * f; acc[k].z += v[i].z * f; acc[k].w += v[i].w * f;
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int idx = tid + k * WARPS * 32, rr = idx / (D / 4), d = idx % (D / 4) * 4, row = row0 + rr;
    if (rr < rows) write_row4<T>(p, qs + row / p.G, kvh * p.G + row % p.G, D, d, acc[k], state[rr * 3 + 1]);
  }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32, RESIDENT<D, NT>)
attention_packed_kernel(const PackedParams p) {
  using B = PackedBlock<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars_mem[WARPS * HALVES];
  __shared__ long long s_scan[WARPS];
  __shared__ int s_req, s_begin;
  __shared__ Way way;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* ring = smem + warp * HALVES * NB * B::BYTES;
  float* merge = reinterpret_cast<float*>(smem + WARPS * HALVES * NB * B::BYTES);
  const uint32_t bars = sm100::smem_u32(bars_mem + warp * HALVES);
  if (lane == 0)
    for (int s = 0; s < HALVES; ++s) sm100::mbar_init(bars + 8 * s, 1);
  sm100::fence_barrier_init();
  sm100::fence_proxy_async();
  pdl_wait();
  pdl_launch();
  // ---- the CTA's first item
  // CTAs that a pair of its own gets: their sum over all pairs is at most N + (P - N)
  auto ctas_of = [&](const Span sp) { return sp.tiles ? (int)min((long long)(sp.tiles + NB - 1) / NB, 1 + (long long)sp.tiles * max(0ll, way.P - way.N) / way.U) : 0; };
  auto pairs_of = [&](const Span sp) { return sp.row_tiles * p.Hkv; };
  // units in the low 40 bits, pairs above
  auto load_of = [&](const Span sp) {
    if (sp.tiles == 0 && sp.row_tiles) atomicExch(p.err, 5);
    return sp.tiles ? (long long)sp.tiles * pairs_of(sp) + ((long long)pairs_of(sp) << 40) : 0ll;
  };
  auto length_of = [&](const Span sp) { return way.own ? ctas_of(sp) : sp.tiles ? sp.tiles + EXTRA : 0; };
  auto line_of = [&](const Span sp) { return (long long)length_of(sp) * pairs_of(sp); };
  auto decide = [&](long long load) {      // the same in every thread
    const long long c = blockIdx.x, U = load & ((1ll << 40) - 1), N = load >> 40, L = U + EXTRA * N;
    const bool own = OWN * N <= gridDim.x;
    const long long P = min((long long)gridDim.x, own ? U : L);
    if (tid == 0 && U) way = Way{L, U, P, N, own ? c : c * L / P, own ? c + 1 : (c + 1) * L / P, (int)min((long long)WHOLE, L / P), own};
    return U > 0 && (own || c < P);
  };
  auto run_in_warp = [&](long long v) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += x;
    }
    return v;
  };
  int r = -1, begin = 0;               // the item's request, and where its line begins, counted from the CTA's share
  if (p.n_reqs <= 32) {                // every warp looks at all of them
    const Span sp = lane < p.n_reqs ? span_of<NT>(p, lane) : Span{0, 0, 0};
    if (!decide(__shfl_sync(0xffffffffu, run_in_warp(load_of(sp)), 31))) return;
    __syncthreads();
    const long long mine = line_of(sp), at = run_in_warp(mine) - mine;
    const unsigned here = __ballot_sync(0xffffffffu, way.first >= at && way.first < at + mine);
    if (here == 0) return;
    r = __ffs(here) - 1;
    begin = (int)(__shfl_sync(0xffffffffu, at, r) - way.first);
  } else {                             // 128 at a time, one a thread
    long long mine = 0, at = 0, line = 0;
    auto scan = [&](int base, auto count) {
      mine = base + tid < p.n_reqs ? count(span_of<NT>(p, base + tid)) : 0;
      const long long u = run_in_warp(mine);
      __syncthreads();
      if (lane == 31) s_scan[warp] = u;
      __syncthreads();
      at = line + u - mine;
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) at += s_scan[w];
        line += s_scan[w];
      }
    };
    for (int base = 0; base < p.n_reqs; base += WARPS * 32) scan(base, load_of);
    if (!decide(line)) return;
    if (tid == 0) s_req = -1;
    line = 0;
    __syncthreads();
    for (int base = 0; base < p.n_reqs; base += WARPS * 32) {
      scan(base, line_of);
      if (way.first >= at && way.first < at + mine) {
        s_req = base + tid;
        s_begin = (int)(at - way.first);
      }
      if (line > way.first) break;
    }
    __syncthreads();
    r = s_req;
    begin = s_begin;
    if (r < 0) return;
  }
  int done = 0;                        // of the CTA's share
  auto next_item = [&](Item& it) {
    const long long P = way.P, L = way.L;
    while (done < way.last - way.first) {
      const Span sp = span_of<NT>(p, r);
      if (done >= begin + line_of(sp)) {
        begin += (int)line_of(sp);
        ++r;
        continue;
      }
      const int each = length_of(sp), pair = (done - begin) / each, i = (done - begin) % each;
      const int blocks = (p.pos0[r] + p.q_start[r + 1] - p.q_start[r] - sp.lo + PACKED_POS - 1) / PACKED_POS;
      it.r = r;
      it.kvh = pair / sp.row_tiles;
      it.rt = pair % sp.row_tiles;
      it.key_lo = sp.lo;
      if (way.own) {
        it.q0 = (int)((long long)i * blocks / each);
        it.q1 = (int)((long long)(i + 1) * blocks / each);
        it.parts = Parts{(int)blockIdx.x - i, each};
        done = 1;
        return true;
      }
      const int after = done - i + each;      // where the pair ends
      if (sp.tiles <= way.whole) {
        done = after;
        if (i > 0) continue;                  // it begins in another CTA's stretch
        it.q0 = 0;
        it.q1 = blocks;
        it.parts = Parts{0, 1};
        return true;
      }
      const long long pair_start = way.first + begin + (long long)pair * each;
      const int t0 = max(0, i - EXTRA), t1 = (int)min((long long)sp.tiles, way.last - pair_start - EXTRA);
      done = min(after, (int)(way.last - way.first));
      if (t0 >= t1) continue;                 // the stretch ends within the pair's EXTRA
      it.q0 = t0 * WARPS;
      it.q1 = min(blocks, t1 * WARPS);
      // the CTAs of the pair's first and last units: the largest k with k L / P <= that unit's place
      const int k0 = (int)(((pair_start + EXTRA + 1) * P - 1) / L), k1 = (int)(((pair_start + each) * P - 1) / L);
      it.parts = Parts{k0, k1 - k0 + 1};
      return true;
    }
    return false;
  };
  // ---- walk the share
  uint32_t turn = 0;      // steps that the warp has run: a step's half of the ring and its barrier's phase follow from its number
  bool failed = false;
  Flow<D> flow;
  Item it, following;
  bool more = next_item(it);
  if (more) flow.begin(p, it, turn, ring, bars);
  while (more) {
    packed_item<T, D, NT>(p, it, flow, ring, bars, turn, merge, failed, [&]() {
      more = next_item(following);
      if (more) flow.begin(p, following, turn, ring, bars);
    });
    it = following;
  }
}

template <typename T, int D, int NT>
int launch_packed(const PackedParams& p, cudaStream_t stream) {
  static_assert(8 * NT * (64 + 3) <= WARPS * 8 * (D + 2), "the parts' factors lie where the warps' sums did");
  constexpr int smem = WARPS * HALVES * NB * PackedBlock<D>::BYTES + WARPS * 8 * (D + 2) * 4;
  static bool configured = false;
  if (!configured) {
    cudaError_t e = cudaFuncSetAttribute(attention_packed_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    FERRUM_CHECK_ARG(e == cudaSuccess, "attention_packed: cannot reserve %d bytes of shared memory: %s", smem, cudaGetErrorString(e));
    configured = true;
  }
  // no more CTAs than the longest requests that the tables can hold have units
  const long long units = (long long)p.n_reqs * p.Hkv * (NT == 1 ? 2 : 1) * (((long long)p.table_width * p.page_size + TILE - 1) / TILE + 1);
  const int ctas = (int)std::min<long long>(RESIDENT<D, NT> * ferrum_sm_count(), units);
  launch_kernel(attention_packed_kernel<T, D, NT>, dim3(ctas), dim3(WARPS * 32), smem, stream, p);
  FERRUM_CHECK_LAUNCH("attention_packed");
  return 0;
}

int most_ctas() { return MAX_RESIDENT * ferrum_sm_count(); }

}  // namespace

FERRUM_API int ferrum_attention_packed_rows() { return PACKED_FEW_ROWS; }

// Floats of workspace that a call needs: two slots a CTA for partials.
FERRUM_API long long ferrum_attention_packed_workspace(int D) { return (long long)most_ctas() * 2 * PART_ROWS * (D + 2); }

// part: workspace of ferrum_attention_packed_workspace(D) floats; counters: n_reqs * Hkv * 2 int32 zeros, which the call leaves zeros.
// Calls that may run at the same time need one of each for themselves.  row_tiles: rows that a pass over a request's keys takes, in tiles of eight (a request of
// more than eight takes two passes with one).
FERRUM_API int ferrum_attention_packed(const void* q, int ldq, void* out, int ldo, int dtype, const void* plane, long long page_stride, int n_pages,
                                       int page_size, const int* block_table, int table_width, const int* q_start, const int* pos0, int n_reqs,
                                       int row_tiles, float* part, long long part_floats, int* counters, int n_counters, int Hq, int Hkv, int D, float scale, int window,
                                       int* err_flag, cudaStream_t stream) {
  FERRUM_CHECK_ARG(Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "attention_packed: bad head counts Hq=%d Hkv=%d", Hq, Hkv);
  FERRUM_CHECK_ARG(D == 64 || D == 128, "attention_packed: a cache in 4 bits has heads of 64 or 128 elements, found %d", D);
  FERRUM_CHECK_ARG(packed_page_ok(page_size) && table_width > 0 && n_pages > 0 && window >= 0 && n_reqs >= 0,
                   "attention_packed: bad sizes (page size %d must be a multiple of %d)", page_size, PACKED_POS);
  FERRUM_CHECK_ARG(row_tiles == 1 || row_tiles == 2, "attention_packed: a pass takes one or two tiles of eight rows, found %d", row_tiles);
  FERRUM_CHECK_ARG(err_flag != nullptr, "attention_packed: the error flag is required");
  FERRUM_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)plane | (uintptr_t)part) & 15) == 0 && ldq % 8 == 0 && ldo % 8 == 0 && page_stride % 16 == 0,
                   "attention_packed: operands must be 16-byte aligned");
  FERRUM_CHECK_ARG(ldq >= Hq * D && ldo >= Hq * D, "attention_packed: rows of %d and %d elements are too short", ldq, ldo);
  FERRUM_CHECK_ARG(part_floats >= ferrum_attention_packed_workspace(D) && n_counters >= (long long)n_reqs * Hkv * 2, "attention_packed: the workspace is too small");
  if (n_reqs == 0) return 0;
  const int G = Hq / Hkv;
  float* part_ml = part + (size_t)most_ctas() * 2 * PART_ROWS * D;
  PackedParams p{q, out, (const uint8_t*)plane, block_table, q_start, pos0, part, part_ml, counters,
                 err_flag, page_stride, ldq, ldo, n_pages, page_size, table_width, (int)std::min<long long>((long long)table_width * page_size, 0x7fffff00), Hq, Hkv, G, window,
                 n_reqs, scale * 1.4426950408889634f};
  const bool narrow = row_tiles == 1;
  FERRUM_DISPATCH_16BIT(dtype, T, {
    if (D == 64) return narrow ? launch_packed<T, 64, 1>(p, stream) : launch_packed<T, 64, 2>(p, stream);
    return narrow ? launch_packed<T, 128, 1>(p, stream) : launch_packed<T, 128, 2>(p, stream);
  });
  return 0;
}
