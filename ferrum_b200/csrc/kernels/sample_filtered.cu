// Next-token draw from given random numbers: temperature, top-k, top-p and min-p, in this order.
//
// Of a row x of logits, with z_i = (x_i - max) / T and w_i = exp(z_i) in 64 bits (NaN logits are left out):
//   top-k   the k largest stay (of equal ones the lower index)
//   top-p   in that order a token stays while the mass of the tokens before it is below p times the mass that top-k left
//   min-p   a token stays if w_i >= min_p (the largest w is 1)
//   draw    the first token in index order at which the running mass of those that stay exceeds u times their whole mass
// T = 0 takes the largest logit.  Masses are whole numbers, w_i rounded to 2^-s with s = 62 - ceil(log2 V): their sums are exact whatever
// their order, and 2^-s (2^-45 at 128 Ki tokens) is far below what a draw's 53 random bits can tell from 0.
//
// Simplest form: a block per row; every threshold by bisection over the logits' bits as ordered integers, a pass over the row each.
// The reference samples greedily only (crates/core-types/src/model.rs:44-62).
#include "common.cuh"

namespace {

typedef unsigned long long u64;

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
  int ld, V, shift;
};

__device__ __forceinline__ u64 block_sum64(u64 v, u64* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) t += red[i];
  return t;
}

__device__ __forceinline__ double weight(uint32_t key, float top, float T) {
  const float x = key_value(key);
  return x == top ? 1.0 : exp(((double)x - (double)top) / (double)T);
}
__device__ __forceinline__ u64 mass_of(double w, int shift) { return __double2ull_rn(w * (double)(1ull << shift)); }

__global__ void __launch_bounds__(1024)
sample_filtered_kernel(const FilterParams p) {
  __shared__ u64 red[32];
  __shared__ int s_id;
  __shared__ u64 s_run[3];
  pdl_launch();
  pdl_wait();
  const int r = p.rows ? p.rows[blockIdx.x] : blockIdx.x, tid = threadIdx.x, V = p.V;
  const float* row = p.logits + (size_t)r * p.ld;
  const float T = p.temperature[blockIdx.x], top_p = p.top_p ? p.top_p[blockIdx.x] : 1.f, min_p = p.min_p ? p.min_p[blockIdx.x] : 0.f;
  const int top_k = p.top_k ? p.top_k[blockIdx.x] : 0;
  auto finish = [&](int id, int code) {
    if (tid == 0) {
      p.out_ids[r] = id;
      if (p.also_to) p.also_to[r] = id;
      if (code) atomicExch(p.err, code);
    }
  };
  if (!(T >= 0.f) || T == INFINITY || !(top_p > 0.f) || !(min_p <= 1.f)) {      // (the same for the whole block)
    finish(-1, 7);
    return;
  }
  uint32_t best = 0;
  for (int i = tid; i < V; i += blockDim.x) best = max(best, order_key(row[i]));
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  __syncthreads();
  if ((tid & 31) == 0) red[tid >> 5] = best;
  __syncthreads();
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) best = max(best, (uint32_t)red[i]);
  if (best == 0) {
    finish(-1, 6);
    return;
  }
  const float top = key_value(best);
  auto count_from = [&](uint32_t key) {
    u64 n = 0;
    for (int i = tid; i < V; i += blockDim.x) n += order_key(row[i]) >= key;
    return block_sum64(n, red);
  };
  uint32_t t_key = 1;          // tokens above t_key stay, of those equal to it the first `ties`
  u64 ties = ~0ull;
  if (T == 0.f) {
    t_key = best;
    ties = 1;
  } else if (top_k > 0 && top_k < V) {
    uint32_t lo = 1, hi = best;      // the largest key that at least top_k tokens reach, or 1
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      if (count_from(mid) >= (u64)top_k) lo = mid; else hi = mid - 1;
    }
    t_key = lo;
    const u64 above = t_key == 0xffffffffu ? 0 : count_from(t_key + 1);
    ties = (u64)top_k > above ? (u64)top_k - above : 0;
  }
  const float Tw = T == 0.f ? 1.f : T;
  auto mass_above = [&](uint32_t key) {       // tokens that stay so far with a key above `key`
    u64 m = 0, n = 0;
    for (int i = tid; i < V; i += blockDim.x) {
      const uint32_t k = order_key(row[i]);
      if (k > key && k > t_key) m += mass_of(weight(k, top, Tw), p.shift);
      if (k > key && k == t_key) ++n;
    }
    m = block_sum64(m, red);
    n = block_sum64(n, red);
    return m + min(n, ties) * mass_of(weight(t_key, top, Tw), p.shift);
  };
  if (T > 0.f && top_p < 1.f) {
    const double target = (double)top_p * (double)mass_above(t_key - 1);
    uint32_t lo = t_key, hi = best;          // the smallest key whose tokens above weigh less than the target
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((double)mass_above(mid) < target) hi = mid; else lo = mid + 1;
    }
    const u64 before = mass_above(lo), each = mass_of(weight(lo, top, Tw), p.shift);
    // of the tokens at the border the i-th stays if before + i * each < target
    u64 stay = ~0ull;
    if (each > 0) {
      const double room = target - (double)before;
      stay = (u64)ceil(room / (double)each);
      while (stay > 0 && (double)(before + (stay - 1) * each) >= target) --stay;
      while ((double)(before + stay * each) < target) ++stay;
    }
    ties = lo == t_key ? min(ties, stay) : stay;
    t_key = lo;
  }
  // the whole mass, then the draw: both in index order, a tile of blockDim tokens at a time
  const int lane = tid & 31, warp = tid >> 5;
  u64 threshold = 0;
  for (int pass = 0; pass < 2; ++pass) {
    u64 run_mass = 0, run_ties = 0;
    if (tid == 0) s_id = V;
    for (int base = 0; base < V; base += blockDim.x) {
      const uint32_t k = base + tid < V ? order_key(row[base + tid]) : 0;
      u64 t = k == t_key;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += v;
      }
      __syncthreads();
      if (lane == 31) red[warp] = t;
      __syncthreads();
      u64 before = run_ties, all = run_ties;
      for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
        if (i < warp) before += red[i];
        all += red[i];
      }
      run_ties = all;
      const bool stays = k != 0 && (k > t_key || (k == t_key && before + t <= ties));
      u64 m = 0;
      if (stays) {
        const double w = weight(k, top, Tw);
        if (!(min_p > 0.f) || w >= (double)min_p) m = mass_of(w, p.shift);
      }
      const u64 mine = m;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 v = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) m += v;
      }
      __syncthreads();
      if (lane == 31) red[warp] = m;
      __syncthreads();
      before = run_mass, all = run_mass;
      for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
        if (i < warp) before += red[i];
        all += red[i];
      }
      run_mass = all;
      if (pass == 1 && mine > 0 && before + m > threshold && before + m - mine <= threshold) s_id = base + tid;
    }
    if (pass == 0) {
      const double u = p.uniform ? p.uniform[blockIdx.x] : 0.0;
      const double x = u > 0.0 ? u * (double)run_mass : 0.0;
      threshold = x >= (double)run_mass ? run_mass - 1 : min((u64)x, run_mass - 1);
    }
  }
  __syncthreads();
  finish(s_id, 0);
}

}  // namespace

FERRUM_API int ferrum_sample_filtered(const float* logits, int ld, int n_rows, int V, const int* rows, const float* temperature, const int* top_k,
                                      const float* top_p, const float* min_p, const double* uniform, int* out_ids, int* also_to, int* err_flag,
                                      cudaStream_t stream) {
  FERRUM_CHECK_ARG(n_rows >= 0 && V > 0 && ld >= V, "sample_filtered: bad sizes rows=%d V=%d ld=%d", n_rows, V, ld);
  FERRUM_CHECK_ARG(temperature && uniform && out_ids && err_flag, "sample_filtered: temperature, uniform, out_ids and the error flag are required");
  if (n_rows == 0) return 0;
  int bits = 0;
  while (bits < 31 && (1ll << bits) < V) ++bits;
  FilterParams p{logits, rows, temperature, top_k, top_p, min_p, uniform, out_ids, also_to, err_flag, ld, V, 62 - bits};
  launch_kernel(sample_filtered_kernel, dim3(n_rows), dim3(V >= 8192 ? 1024 : 256), 0, stream, p);
  FERRUM_CHECK_LAUNCH("sample_filtered");
  return 0;
}
