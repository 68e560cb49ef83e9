// Next-token draw from given random numbers: temperature, top-k, top-p and min-p, in this order.
//
// Of a row x of logits, with z_i = (x_i - max) / T and w_i = exp(z_i) (NaN logits are left out):
//   top-k   the k largest stay (of equal ones the lower index)
//   top-p   in that order a token stays while the mass of the tokens before it is below p times the mass that top-k left
//   min-p   a token stays if w_i >= min_p (the largest w is 1)
//   draw    the first token in index order at which the running mass of those that stay exceeds u times their whole mass
// T = 0 takes the largest logit.  Masses are whole numbers, w_i rounded to 2^-s with s = min(45, 62 - ceil(log2 V)): their sums are exact
// whatever their order, and 2^-45 is far below what a row's sum of 32-bit weights could tell apart.
//
// A cluster of CTAs holds a row's logits in its shared memory, as integers of the same order; a warp owns a run of them.  Where top-k or
// top-p cuts is found by histograms: 2,048 bins of equal width below the maximum, then the range of keys in the bin that holds the
// cut, cut into 2,048 again, until that bin holds a single key (one or two histograms for logits of any real model, four at
// most).  Each CTA counts its slice; of the bins' sums over the cluster each CTA makes its share.  What lies in the bin of the cut or
// above it is listed on the way, in index order, and all that follows reads the lists (where a warp's share outgrows its list,
// the slice again).  Where the first histogram leaves no more than 1,024 tokens, the usual case, one CTA sorts those and does the rest alone.  Of equal keys at the cut the first in index order stay: a threshold is a key and an index.
//
// What bounds it is neither bytes (64 rows of 128,256 logits are read once: 5 us at 6.5 TB/s) nor arithmetic but the chain of passes over shared memory and
// of cluster barriers between them, and for many rows that their clusters do not all find room at a time.  B200, 128,256 logits, in a CUDA graph: one row
// with top-k 50 19.5 us, with top-p alone 29, unfiltered 11; 8 rows with top-k 23; 64 rows with top-k 59, unfiltered 52, each with filters of its own 83 (0.4 TB/s).
//
// The reference samples greedily only (crates/core-types/src/model.rs:44-62).
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int BINS = 2048;
constexpr int MAX_CLUSTER = 16;
constexpr int THREADS = 512;         // two CTAs an SM
constexpr int WARPS = THREADS / 32;
constexpr int SEGMENTS = 2;         // parts of a warp's run whose masses are kept for the draw
constexpr int LIST = 1024;          // listed tokens of a CTA, LIST / warps of a warp
constexpr int MOST_BINS = BINS / THREADS;      // bins of a thread's share
constexpr int FEW = 1024;           // tokens that one CTA sorts

// Order-preserving integer of a logit; 0 stands for NaN, which comes after everything and is never kept.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);      // (-0 and 0 are equal)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct FilterParams {
  const float* logits;
  const int* rows;                  // null: row r of the launch is row r of the logits
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const double* uniform;
  int* out_ids;
  int* also_to;
  int* err;
  int ld, V, per, shift, held;      // per: logits of a CTA's slice; held: rows that there are
};

// A token stays while (key, index) comes no later than the threshold: larger keys first, then lower indices.
struct Cut {
  uint32_t key;
  int index;
  __device__ __forceinline__ bool stays(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};

__device__ __forceinline__ uint32_t peer(uint32_t local, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
__device__ __forceinline__ u64 load_peer(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void store_peer(uint32_t addr, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory"); }
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Shared {
  union {
    u64 hist[BINS];
    struct {
      u64 order[FEW], mass[FEW];    // the first CTA's: (key, ~index) of the tokens at or above the cut, and their masses
    };
  };
  unsigned few;                     // how many there are
  u64 exchange[4][2][MAX_CLUSTER];
  u64 warp[32][2];
  u64 segment[WARPS][SEGMENTS];
  u64 found[2];
  uint32_t list_key[LIST];
  int list_index[LIST];
  double powers[64];                // 2^(j / 64)
};

// What a first histogram has told: the bin of the cut (none: -1), the sum of what lies above it, and the limit.
struct Border {
  int bin;
  u64 before;
  double limit;
};

// The CTA's view of its row.
template <bool RESIDENT>
struct Row {
  const FilterParams& p;
  Shared& sh;
  const uint32_t* keys;             // the slice in shared memory, or
  const float* row;                 // in global memory
  int rank, n_ctas, lo;             // the slice's first logit
  int e0, e1;                       // the warp's run: entries e0 .. e1 - 1 of the slice, or of the lists
  bool listed;
  int turn;                         // exchanges so far
  uint32_t best;
  float top;
  double inv_t;

  __device__ __forceinline__ uint32_t key(int e) const { return listed ? sh.list_key[e] : RESIDENT ? keys[e] : order_key(row[lo + e]); }
  __device__ __forceinline__ int index(int e) const { return listed ? sh.list_index[e] : lo + e; }

  // w * 2^shift of a key, not rounded.  exp by 2^(n / 64) from a table and the series of the rest (below 2^-7 in size: the sixth term is
  // 3e-17 of the sum); what is below 2^-1 after the scaling rounds to 0 whatever its value.
  // Without a branch, so that several weights are on their way at a time.
  __device__ __forceinline__ double scaled_weight(uint32_t k) const {
    const double exact = ((double)key_value(k) - (double)top) * inv_t * 92.332482616893656877;      // 64 log2(e)
    const double y = fmax(exact, -3000.0);                        // (-infinity, and the NaN of two infinities)
    const double t = y + 6755399441055744.0;                       // 1.5 * 2^52: the nearest whole number in the low bits
    const int n = __double2loint(t);
    const double q = (y - (t - 6755399441055744.0)) * 0.010830424696249145347;               // ln(2) / 64
    const double s = fma(q, fma(q, fma(q, fma(q, fma(q, 1.0 / 120.0, 1.0 / 24.0), 1.0 / 6.0), 0.5), 1.0), 1.0);
    const double v = sh.powers[n & 63] * s;
    const double w = __hiloint2double(__double2hiint(v) + (((n >> 6) + p.shift) << 20), __double2loint(v));
    return k == best ? (double)(1ull << p.shift) : exact > -3000.0 ? w : 0.0;
  }
  static __device__ __forceinline__ u64 whole(double v) { return (u64)__double_as_longlong(v + 4503599627370496.0) & 0xfffffffffffffull; }      // (v below 2^51)
  __device__ __forceinline__ u64 mass(uint32_t k) const { return whole(scaled_weight(k)); }

  // hist[bin_of(k)] += 1 or (MASS) the mass of k, for the tokens of the warp's run that wanted(key, entry) names.
  template <bool MASS, typename Wanted, typename Bin>
  __device__ __forceinline__ void fill_histogram(Wanted wanted, Bin bin_of) {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < BINS; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    constexpr int AT_ONCE = 4;
    for (int e = e0 + lane; e - lane < e1; e += 32 * AT_ONCE) {
      uint32_t k[AT_ONCE];
      u64 v[AT_ONCE];
      bool any = false;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int at = e + 32 * i;
        k[i] = at < e1 ? key(at) : 0;
        if (k[i] && !wanted(k[i], at)) k[i] = 0;
        any |= k[i] != 0;
      }
      if (!__any_sync(0xffffffffu, any)) continue;
      if (MASS) {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) v[i] = mass(k[i]);
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        if (k[i] == 0) continue;
        unsigned* half = reinterpret_cast<unsigned*>(&sh.hist[bin_of(k[i])]);      // (a 64-bit addition by two of 32 bits, the second hardly ever made)
        if (MASS) {
          const unsigned low = (unsigned)v[i];
          if (v[i] == 0) continue;
          const unsigned old = atomicAdd(half, low), high = (unsigned)(v[i] >> 32) + (old + low < old ? 1 : 0);
          if (high) atomicAdd(half + 1, high);
        } else {
          atomicAdd(half, 1u);
        }
      }
    }
  }

  // Sums (or maxima of) two numbers over the block, then hands them to every CTA; afterwards exchange[..][0 or 1][c] holds CTA c's.
  template <bool MAXIMA>
  __device__ __forceinline__ const u64 (&gather(u64 a, u64 b))[2][MAX_CLUSTER] {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 x = __shfl_xor_sync(0xffffffffu, a, o), y = __shfl_xor_sync(0xffffffffu, b, o);
      a = MAXIMA ? max(a, x) : a + x;
      b = MAXIMA ? max(b, y) : b + y;
    }
    __syncthreads();
    if (lane == 0) sh.warp[warp][0] = a, sh.warp[warp][1] = b;
    __syncthreads();
    u64(&ex)[2][MAX_CLUSTER] = sh.exchange[turn++ & 3];
    if (warp == 0) {
      a = lane < WARPS ? sh.warp[lane][0] : 0;
      b = lane < WARPS ? sh.warp[lane][1] : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const u64 x = __shfl_xor_sync(0xffffffffu, a, o), y = __shfl_xor_sync(0xffffffffu, b, o);
        a = MAXIMA ? max(a, x) : a + x;
        b = MAXIMA ? max(b, y) : b + y;
      }
      if (lane < n_ctas) {
        store_peer(peer((uint32_t)__cvta_generic_to_shared(&ex[0][rank]), lane), a);
        store_peer(peer((uint32_t)__cvta_generic_to_shared(&ex[1][rank]), lane), b);
      }
    }
    cluster_sync();
    return ex;
  }
  // One thread of one CTA tells every CTA two numbers (the others pass `mine` false).
  __device__ __forceinline__ void tell(bool mine, u64 a, u64 b) {
    u64(&ex)[2][MAX_CLUSTER] = sh.exchange[turn++ & 3];
    if (mine)
      for (int c = 0; c < n_ctas; ++c) {
        store_peer(peer((uint32_t)__cvta_generic_to_shared(&ex[0][0]), c), a);
        store_peer(peer((uint32_t)__cvta_generic_to_shared(&ex[1][0]), c), b);
      }
    cluster_sync();
    __syncthreads();
    if (threadIdx.x == 0) sh.found[0] = ex[0][0], sh.found[1] = ex[1][0];
    __syncthreads();
  }

  // Running sums of mass[0 .. size - 1] in place (size a power of two, at least 32 and at most 2 * blockDim).
  __device__ __forceinline__ void run_sums(int size) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = size / 32;
    __syncthreads();
    for (int w = warp; w < chunks; w += WARPS) {
      u64 v = sh.mass[w * 32 + lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      sh.mass[w * 32 + lane] = v;
    }
    __syncthreads();
    if (warp == 0) {                // the chunks' totals, one a lane
      u64 v = lane < chunks ? sh.mass[lane * 32 + 31] : 0;
      const u64 own = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      sh.warp[lane][0] = v - own;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += THREADS) sh.mass[i] += sh.warp[i >> 5][0];
    __syncthreads();
  }
  // order[0 .. size - 1], the largest first.
  __device__ __forceinline__ void sort_down(int size) {
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int t = threadIdx.x; t < size / 2; t += THREADS) {
          const int i = 2 * t - (t & (j - 1));      // the lower of the pair (i, i + j)
          const u64 a = sh.order[i], b = sh.order[i + j];
          if ((a < b) == ((i & k) == 0)) sh.order[i] = b, sh.order[i + j] = a;
        }
      }
    __syncthreads();
  }

  // Rows whose cut leaves few tokens: one histogram, and the tokens of the bins down to the one that holds the cut go to the first CTA, which sorts
  // them and does the rest.  BY_MASS: no top-k, so that the cut is top-p's.  False (for all CTAs alike): there are more than FEW of them; `known` is what
  // the histogram told then.
  template <bool BY_MASS>
  __device__ __forceinline__ bool draw_of_few(int top_k, float top_p, double min_w, double u, float range, int out, Border& known) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!(isfinite(top) && isfinite(range))) return false;
    const float scale = (float)BINS / range;
    auto bin_of = [&](uint32_t k) { return min(BINS - 1, (int)((top - key_value(k)) * scale)); };
    fill_histogram<BY_MASS>([](uint32_t, int) { return true; }, bin_of);
    cluster_sync();
    u64 mine[MOST_BINS], own, all, at;
    int b0, each;
    bins_of_cluster(mine, own, all, at, b0, each);
    const double limit = BY_MASS ? (double)top_p * (double)all : (double)top_k;
    u64 best_bin = 0, best_at = 0;
#pragma unroll
    for (int j = 0; j < MOST_BINS; ++j) {
      if (j < each && mine[j] && (double)at < limit) best_bin = b0 + j + 1, best_at = at;
      at += mine[j];
    }
    const u64(&e2)[2][MAX_CLUSTER] = gather<true>(best_bin, best_at);
    int border = 0;
    u64 before = 0;
    for (int c = 0; c < n_ctas; ++c) border = max(border, (int)e2[0][c]), before = max(before, e2[1][c]);
    known = Border{border - 1, before, limit};
    // (the bins are read: their place is free)
    unsigned count = 0;
#pragma unroll 4
    for (int e = e0 + lane; e < e1; e += 32) {
      const uint32_t k = key(e);
      count += k != 0 && bin_of(k) < border;
    }
    const unsigned total = __reduce_add_sync(0xffffffffu, count);
    if (total) {
      unsigned base = 0;
      if (lane == 0)
        asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;"
                     : "=r"(base) : "r"(peer((uint32_t)__cvta_generic_to_shared(&sh.few), 0)), "r"(total) : "memory");
      base = __shfl_sync(0xffffffffu, base, 0);
      if (base + total <= FEW)
        for (int e = e0 + lane; e - lane < e1; e += 32) {
          const uint32_t k = e < e1 ? key(e) : 0;
          const bool goes = k != 0 && bin_of(k) < border;
          const unsigned hit = __ballot_sync(0xffffffffu, goes);
          if (goes)
            store_peer(peer((uint32_t)__cvta_generic_to_shared(&sh.order[base + __popc(hit & ((1u << lane) - 1))]), 0), (u64)k << 32 | (uint32_t)~index(e));
          base += __popc(hit);
        }
    }
    cluster_sync();
    unsigned n;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(peer((uint32_t)__cvta_generic_to_shared(&sh.few), 0)) : "memory");
    cluster_sync();                 // (read before the first CTA goes on, or leaves)
    if (n > FEW) return false;
    if (rank != 0) return true;
    int size = 32;
    while (size < (int)n) size <<= 1;
    for (int i = tid; i < size; i += THREADS)
      if (i >= (int)n) sh.order[i] = 0;
    sort_down(size);
    auto weigh = [&](int i) { return i < (int)n ? scaled_weight((uint32_t)(sh.order[i] >> 32)) : 0.0; };
    for (int i = tid; i < size; i += THREADS) sh.mass[i] = whole(weigh(i));
    run_sums(size);
    const int n_k = BY_MASS ? (int)n : min((int)n, top_k);
    const double part = BY_MASS ? limit : top_p < 1.f ? (double)top_p * (double)sh.mass[n_k - 1] : INFINITY;
    // what stays are the first so many
    int stays = 0;
    for (int i = tid; i < n_k; i += THREADS)
      if ((i == 0 || (double)sh.mass[i - 1] < part) && weigh(i) >= min_w) stays = i + 1;
    stays = __reduce_max_sync(0xffffffffu, stays);
    __syncthreads();
    if (lane == 0) sh.warp[warp][1] = stays;
    __syncthreads();
    for (int w = 0; w < WARPS; ++w) stays = max(stays, (int)sh.warp[w][1]);
    const u64 sum = sh.mass[stays - 1];
    const double x = u > 0.0 ? u * (double)sum : 0.0;
    const u64 threshold = x >= (double)sum ? sum - 1 : min((u64)x, sum - 1);
    // in index order: (~index, key) from the largest down
    size = 32;
    while (size < stays) size <<= 1;
    for (int i = tid; i < size; i += THREADS) {
      const u64 v = sh.order[i];
      sh.order[i] = i < stays ? v << 32 | v >> 32 : 0;
    }
    sort_down(size);
    for (int i = tid; i < size; i += THREADS) sh.mass[i] = i < stays ? mass((uint32_t)sh.order[i]) : 0;
    run_sums(size);
    for (int i = tid; i < stays; i += THREADS)
      if (threshold < sh.mass[i] && (i == 0 || threshold >= sh.mass[i - 1])) {
        const int id = (int)~(uint32_t)(sh.order[i] >> 32);
        p.out_ids[out] = id;
        if (p.also_to) p.also_to[out] = id;
      }
    return true;
  }

  // The CTA's share of the histogram's bins, `each` from b0 on for the first threads: their sums over the cluster (mine, zeros beyond), what lies in the
  // bins before them (at) and in all (all).  All threads of the cluster call it behind the barrier that ends the counting.
  __device__ __forceinline__ void bins_of_cluster(u64 (&mine)[MOST_BINS], u64& own, u64& all, u64& at, int& b0, int& each) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, share = BINS / n_ctas;
    each = max(1, share / THREADS);
    b0 = rank * share + tid * each;
    const bool has = tid * each < share;
    u64 run = 0;
#pragma unroll
    for (int j = 0; j < MOST_BINS; ++j) {
      mine[j] = 0;
      if (has && j < each) {
        const uint32_t a = (uint32_t)__cvta_generic_to_shared(&sh.hist[b0 + j]);
#pragma unroll 8
        for (int c = 0; c < n_ctas; ++c) mine[j] += load_peer(peer(a, c));
      }
      run += mine[j];
    }
    own = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += v;
    }
    const u64(&ex)[2][MAX_CLUSTER] = gather<false>(own, 0);
    // (gather's sums went over sh.warp; the warps' own totals for the running sums follow in it)
    __syncthreads();
    if (lane == 31) sh.warp[warp][0] = run;
    __syncthreads();
    at = run - own;
    all = 0;
    for (int c = 0; c < n_ctas; ++c) {
      if (c < rank) at += ex[0][c];
      all += ex[0][c];
    }
    if (has)
      for (int w = 0; w < warp; ++w) at += sh.warp[w][0];
  }

  // Where a limit cuts: of the tokens that `cut` lets stay, ordered, a token stays while the sum of what comes before it is below the limit;
  // a token counts 1, the limit is `limit` itself, or (MASS) a token counts its mass and the limit is that part of all of it.  range: how
  // far below the maximum the logits go that count (at least).
  template <bool MASS>
  __device__ __forceinline__ Cut find(const Cut cut, double limit, float range, Border known = Border{-1, 0, 0.0}) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t lo_key = 1, hi_key = best;
    u64 before = 0;
    bool whole_known = !MASS;
    // the first histogram's bins are of equal width below the maximum, where that is a finite number
    bool linear = isfinite(top) && isfinite(range);
    const float scale = (float)BINS / range;
    while (lo_key != hi_key) {
      const int bits = 32 - __clz(hi_key - lo_key), down = max(0, bits - 11);
      auto bin_of = [&](uint32_t k) {
        if (!linear) return (int)((hi_key - k) >> down);
        return min(BINS - 1, (int)((top - key_value(k)) * scale));
      };
      int border;
      if (known.bin >= 0) {         // (a first histogram was made before)
        border = known.bin;
        before = known.before;
        limit = known.limit;
        whole_known = true;
        known.bin = -1;
      } else {
        fill_histogram<MASS>([&](uint32_t k, int e) { return k >= lo_key && k <= hi_key && cut.stays(k, index(e)); }, bin_of);
        cluster_sync();
        u64 mine[MOST_BINS], own, all, at;
        int b0, each;
        bins_of_cluster(mine, own, all, at, b0, each);
        at += before;
        if (!whole_known) limit *= (double)all;
        whole_known = true;
        // the last bin with something in it whose predecessors stay below the limit
        u64 best_bin = 0, best_at = 0;
#pragma unroll
        for (int j = 0; j < MOST_BINS; ++j) {
          if (j < each && mine[j] && (double)at < limit) best_bin = b0 + j + 1, best_at = at;
          at += mine[j];
        }
        // bins and their sums rise together: the largest of each belong together
        const u64(&e2)[2][MAX_CLUSTER] = gather<true>(best_bin, best_at);
        u64 bin = 0;
        before = 0;
        for (int c = 0; c < n_ctas; ++c) bin = max(bin, e2[0][c]), before = max(before, e2[1][c]);
        border = (int)bin - 1;
      }
      // the range of the keys in that bin, for the next histogram; and the lists of what lies in it or above
      uint32_t a = 0, b = 0;        // maximum of ~key and of key
      const int most = LIST / WARPS;
      int count = 0;
#pragma unroll 4
      for (int e = e0 + lane; e - lane < e1; e += 32) {
        const uint32_t k = e < e1 ? key(e) : 0;
        const bool fits = k >= lo_key && cut.stays(k, e < e1 ? index(e) : 0);
        const int its = fits && k <= hi_key ? bin_of(k) : -1;
        if (its == border && !(MASS && mass(k) == 0)) {
          a = max(a, ~k);
          b = max(b, k);
        }
        if (!listed) {
          const unsigned hit = __ballot_sync(0xffffffffu, fits && its <= border);
          if (hit) {
            const int slot = count + __popc(hit & ((1u << lane) - 1));
            if ((hit >> lane & 1) && slot < most) {
              sh.list_key[warp * most + slot] = k;
              sh.list_index[warp * most + slot] = index(e);
            }
            count += __popc(hit);
          }
        }
      }
      const u64(&e3)[2][MAX_CLUSTER] = gather<true>((u64)(count > most) << 32 | a, b);
      a = b = 0;
      bool fit = !listed;
      for (int c = 0; c < n_ctas; ++c) {
        a = max(a, (uint32_t)e3[0][c]);
        b = max(b, (uint32_t)e3[1][c]);
        fit &= e3[0][c] >> 32 == 0;
      }
      if (!fit && !listed) {        // (the flag hid a CTA's range: once more without it)
        uint32_t a2 = 0;
        for (int e = e0 + lane; e < e1; e += 32) {
          const uint32_t k = key(e);
          if (k >= lo_key && k <= hi_key && cut.stays(k, index(e)) && bin_of(k) == border && !(MASS && mass(k) == 0)) a2 = max(a2, ~k);
        }
        const u64(&e4)[2][MAX_CLUSTER] = gather<true>(a2, 0);
        a = 0;
        for (int c = 0; c < n_ctas; ++c) a = max(a, (uint32_t)e4[0][c]);
      }
      if (fit) {
        __syncwarp();
        listed = true;
        e0 = warp * most;
        e1 = e0 + count;
      }
      lo_key = ~a;
      hi_key = b;
      linear = false;
    }
    // of the tokens equal to the key at the cut the i-th stays if before + i * one < limit
    const u64 one = MASS ? mass(lo_key) : 1;
    u64 stay = (u64)ceil(fmax(0.0, limit - (double)before) / (double)max(one, 1ull));
    while (stay > 0 && (double)(before + (stay - 1) * one) >= limit) --stay;
    return first_of(lo_key, cut, max(stay, 1ull));
  }

  // The cut behind the stay-th token (counted from 1, in index order) with this key that `cut` lets stay.
  __device__ __forceinline__ Cut first_of(uint32_t key_at, const Cut cut, u64 stay) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned count = 0;
#pragma unroll 4
    for (int e = e0 + lane; e < e1; e += 32) count += key(e) == key_at && cut.stays(key_at, index(e));
    const unsigned total = __reduce_add_sync(0xffffffffu, count);
    const u64(&ex)[2][MAX_CLUSTER] = gather<false>(count, 0);
    u64 all = 0, ahead = 0;
    for (int c = 0; c < n_ctas; ++c) {
      if (c < rank) ahead += ex[0][c];
      all += ex[0][c];
    }
    if (stay >= all) return Cut{key_at, cut.key == key_at ? cut.index : 0x7fffffff};
    __syncthreads();
    if (lane == 0) sh.warp[warp][0] = total;
    __syncthreads();
    for (int w = 0; w < warp; ++w) ahead += sh.warp[w][0];
    bool mine = false;
    int found = 0;
    if (ahead < stay && stay <= ahead + total)
      for (int e = e0 + lane; e - lane < e1; e += 32) {
        const unsigned hit = __ballot_sync(0xffffffffu, e < e1 && key(e) == key_at && cut.stays(key_at, index(e)));
        const u64 here = __popc(hit);
        if (ahead + here >= stay) {
          const int nth = (int)(stay - ahead);      // the nth set bit of hit
          mine = (hit >> lane & 1) && __popc(hit & ((2u << lane) - 1)) == nth;
          if (mine) found = index(e);
          break;
        }
        ahead += here;
      }
    tell(mine, (u64)found, 0);
    return Cut{key_at, (int)sh.found[0]};
  }

  // The draw from the tokens that the cut lets stay and that weigh min_w at least.
  __device__ __forceinline__ void draw(const Cut cut, double min_w, double u, int out) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rows = (e1 - e0 + 31) / 32;
    // the masses of entries of the lines r .. r + AT_ONCE - 1 (of 32) before `end`; false: none has any
    constexpr int AT_ONCE = 4;
    auto masses = [&](int r, int end, u64 (&m)[AT_ONCE]) {
      uint32_t k[AT_ONCE];
      bool any = false;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int e = e0 + (r + i) * 32 + lane;
        k[i] = r + i < end && e < e1 ? key(e) : 0;
        if (k[i] && !cut.stays(k[i], index(e))) k[i] = 0;
        any |= k[i] != 0;
      }
      if (!__any_sync(0xffffffffu, any)) return false;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const double v = scaled_weight(k[i]);
        m[i] = k[i] && v >= min_w ? whole(v) : 0;
      }
      return true;
    };
    u64 sum = 0;
    for (int s = 0; s < SEGMENTS; ++s) {
      u64 part = 0, m[AT_ONCE];
      const int end = rows * (s + 1) / SEGMENTS;
      for (int r = rows * s / SEGMENTS; r < end; r += AT_ONCE)
        if (masses(r, end, m)) part += m[0] + m[1] + m[2] + m[3];
      sum += part;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) sh.segment[warp][s] = part;
    }
    const u64(&ex)[2][MAX_CLUSTER] = gather<false>(sum, 0);
    u64 all = 0, at = 0;
    for (int c = 0; c < n_ctas; ++c) {
      if (c < rank) at += ex[0][c];
      all += ex[0][c];
    }
    const double x = u > 0.0 ? u * (double)all : 0.0;
    const u64 threshold = x >= (double)all ? all - 1 : min((u64)x, all - 1);
    if (threshold < at || threshold >= at + ex[0][rank]) return;
    for (int w = 0; w < warp; ++w)
      for (int s = 0; s < SEGMENTS; ++s) at += sh.segment[w][s];
    for (int s = 0; s < SEGMENTS; ++s) {
      const u64 part = sh.segment[warp][s];
      if (threshold >= at && threshold < at + part) {
        const int end = rows * (s + 1) / SEGMENTS;
        u64 m[AT_ONCE];
        for (int r = rows * s / SEGMENTS; r < end; r += AT_ONCE) {
          if (!masses(r, end, m)) continue;
#pragma unroll
          for (int i = 0; i < AT_ONCE; ++i) {
            u64 run = m[i];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const u64 v = __shfl_up_sync(0xffffffffu, run, o);
              if (lane >= o) run += v;
            }
            if (threshold >= at + run - m[i] && threshold < at + run) {
              const int id = index(e0 + (r + i) * 32 + lane);
              p.out_ids[out] = id;
              if (p.also_to) p.also_to[out] = id;
            }
            at += __shfl_sync(0xffffffffu, run, 31);
          }
        }
        return;
      }
      at += part;
    }
  }
};

template <bool RESIDENT>
__global__ void __launch_bounds__(THREADS, 2)
sample_filtered_kernel(const FilterParams p) {
  extern __shared__ __align__(16) uint32_t slice[];
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  if (tid == 0) sh.few = 0;
  if (tid < 64) sh.powers[tid] = exp2((double)tid / 64.0);
  // a CTA's shared memory may be written by a peer only once the CTA is known to run
  cluster_sync();
  pdl_wait();
  pdl_launch();
  const int q = blockIdx.x, r = p.rows ? p.rows[q] : q, rank = blockIdx.y;
  if (r < 0 || r >= p.held) {       // (the same for the whole cluster)
    if (tid == 0 && rank == 0) atomicExch(p.err, 7);
    return;
  }
  const float* row = p.logits + (size_t)r * p.ld;
  const float T = p.temperature[q], top_p = p.top_p ? p.top_p[q] : 1.f, min_p = p.min_p ? p.min_p[q] : 0.f;
  const int top_k = p.top_k ? p.top_k[q] : 0, lo = min(p.V, rank * p.per), n = min(p.V, lo + p.per) - lo;
  auto refuse = [&](int code) {
    if (tid == 0 && rank == 0) {
      p.out_ids[r] = -1;
      if (p.also_to) p.also_to[r] = -1;
      atomicExch(p.err, code);
    }
  };
  if (!(T >= 0.f) || T == INFINITY || !(top_p > 0.f && top_p <= 1.f) || !(min_p <= 1.f)) {      // (the same for the whole cluster)
    refuse(7);
    return;
  }
  // ---- the slice, its largest key and its smallest of a finite logit
  uint32_t most = 0, least_finite = ~0u;
  auto take = [&](float x) {
    const uint32_t k = order_key(x);
    most = max(most, k);
    if (k > 0x007fffffu) least_finite = min(least_finite, k);      // (0x007fffff: minus infinity)
    return k;
  };
  const int quads = ((uintptr_t)(row + lo) & 15) == 0 ? n / 4 : 0;
#pragma unroll 4
  for (int i = tid; i < quads; i += THREADS) {
    const float4 x = reinterpret_cast<const float4*>(row + lo)[i];
    const uint4 k = make_uint4(take(x.x), take(x.y), take(x.z), take(x.w));
    if (RESIDENT) reinterpret_cast<uint4*>(slice)[i] = k;
  }
#pragma unroll 8
  for (int i = quads * 4 + tid; i < n; i += THREADS) {
    const uint32_t k = take(row[lo + i]);
    if (RESIDENT) slice[i] = k;
  }
  const int lines = (n + 31) / 32;
  Row<RESIDENT> w{p, sh, slice, row, rank, (int)gridDim.y, lo, (int)((long long)(tid >> 5) * lines / WARPS) * 32,
                  min(n, (int)((long long)((tid >> 5) + 1) * lines / WARPS) * 32), false, 0, 0, 0.f, 0.0};
  const u64(&ex)[2][MAX_CLUSTER] = w.template gather<true>(most, (uint32_t)~least_finite);
  for (int c = 0; c < w.n_ctas; ++c) {
    w.best = max(w.best, (uint32_t)ex[0][c]);
    least_finite = min(least_finite, ~(uint32_t)ex[1][c]);
  }
  if (w.best == 0) {
    refuse(6);
    return;
  }
  w.top = key_value(w.best);
  Cut cut{1, 0x7fffffff};
  if (T == 0.f) {
    cut = w.first_of(w.best, cut, 1);
    w.draw(Cut{w.best, cut.index}, 0.0, 0.0, r);
    cluster_sync();
    return;
  }
  w.inv_t = 1.0 / (double)T;
  const float range = least_finite == ~0u ? INFINITY : w.top - key_value(least_finite);
  // (a token further below the maximum than (shift + 1) ln 2 temperatures has no mass)
  const float mass_range = fminf(range, (float)(p.shift + 1) * 0.6931472f * T);
  const double min_w = min_p > 0.f ? (double)min_p * (double)(1ull << p.shift) : 0.0, u = p.uniform[q];
  const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.f;
  Border known{-1, 0, 0.0};
  if (by_k ? top_k <= FEW && w.template draw_of_few<false>(top_k, top_p, min_w, u, range, r, known)
           : by_p && w.template draw_of_few<true>(top_k, top_p, min_w, u, mass_range, r, known))
    return;
  if (by_k) cut = w.template find<false>(cut, (double)top_k, range, known);
  if (by_p) cut = w.template find<true>(cut, (double)top_p, mass_range, by_k ? Border{-1, 0, 0.0} : known);
  w.draw(cut, min_w, u, r);
  cluster_sync();                   // (no CTA leaves while a peer may still reach into its shared memory)
}

// The most logits that a CTA keeps in its shared memory; a row of more than MAX_CLUSTER times that is read from global memory every time.
constexpr int MOST_RESIDENT = 45 * 1024;

template <bool RESIDENT>
int launch_sample(const FilterParams& p, int n_rows, int ctas, cudaStream_t stream) {
  const int smem = RESIDENT ? p.per * 4 : 0;
  static bool configured = false;
  if (!configured) {                  // (for the largest slice there is: calls of other threads ask for the same)
    constexpr int most = RESIDENT ? MOST_RESIDENT * 4 : 0;
    cudaError_t e = cudaFuncSetAttribute(sample_filtered_kernel<RESIDENT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_filtered_kernel<RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    FERRUM_CHECK_ARG(e == cudaSuccess, "sample_filtered: cannot reserve %d bytes of shared memory: %s", most, cudaGetErrorString(e));
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(n_rows, ctas);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = ctas;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ferrum_dependent_launch_enabled() ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, sample_filtered_kernel<RESIDENT>, p);
  FERRUM_CHECK_ARG(e == cudaSuccess, "sample_filtered: launch failed: %s", cudaGetErrorString(e));
  FERRUM_CHECK_LAUNCH("sample_filtered");
  return 0;
}

// CTAs of a row.  What does not find room waits for a whole row: an SM holds two CTAs whose slices are of up to 16,384 logits or so, and clusters of 16 go
// onto few SMs at a time.  B200, top-k 50 and top-p 0.9, us with 1 / 4 / 8 / 16 CTAs (-: not measured):
//   8,192 logits, 8 rows 18 / - / 19 / -, 64 rows 18 / - / 34 / -
//   16,384: 8 rows 23 / - / 15 / 19, 32 rows 22 / 17 / 23 / -, 64 rows 23 / 20 / 36 / -
//   65,536: 4 rows - / - / 18.0 / 17.4, 8 rows - / - / 18 / 21, 16 rows - / 23 / 21 / 30, 32 rows - / 25 / 28 / -, 64 rows - / 29 / 46 / -
//   128,256: 4 rows - / - / 23 / 20, 8 rows - / - / 23 / 24, 16 rows - / 32 / 28 / 35, 64 rows - / 63 / 60 / -; top-p alone at a temperature of 1.3,
//   where the bins above the cut hold too many to list, 1 row - / - / 59 / 41, 64 rows - / 203 / 163 / -
// (CTAs of 1,024 threads, one an SM: 1 row of 128,256 23 instead of 20, 16 rows 40 instead of 28.)
int ctas_of(int n_rows, int V) {
  if (V < 16384) return 1;
  if (n_rows <= 4 && V >= 65536) return MAX_CLUSTER;
  return n_rows > 16 && V <= 65536 ? 4 : 8;
}

}  // namespace

// held: rows of the logits, of out_ids and of also_to; a row named in `rows` beyond them is left out and raises error 7.
FERRUM_API int ferrum_sample_filtered(const float* logits, int ld, int held, int n_rows, int V, const int* rows, const float* temperature, const int* top_k,
                                      const float* top_p, const float* min_p, const double* uniform, int* out_ids, int* also_to, int* err_flag,
                                      cudaStream_t stream) {
  FERRUM_CHECK_ARG(n_rows >= 0 && V > 0 && ld >= V && held >= 0, "sample_filtered: bad sizes rows=%d V=%d ld=%d", n_rows, V, ld);
  FERRUM_CHECK_ARG(temperature && uniform && out_ids && err_flag, "sample_filtered: temperature, uniform, out_ids and the error flag are required");
  if (n_rows == 0) return 0;
  int bits = 0;
  while (bits < 31 && (1ll << bits) < V) ++bits;
  const int ctas = ctas_of(n_rows, V);
  FilterParams p{logits, rows, temperature, top_k, top_p, min_p, uniform, out_ids, also_to, err_flag, ld, V, (V + ctas - 1) / ctas, bits > 17 ? 62 - bits : 45, held};
  if (p.per <= MOST_RESIDENT) return launch_sample<true>(p, n_rows, ctas, stream);
  return launch_sample<false>(p, n_rows, ctas, stream);
}
