// Writing a cache held in 4 bits (packed_cache.cuh has the layout), and bringing pages back to 16 bits.
//
// The write turns the queries and keys by the rotary table and quantises keys and values group by group of 64 elements:
//   lo, hi = min, max;   step = r16(hi f - lo f), f = 1/15 in float32;   middle = r16(lo + 8 step);   code = clamp(rint((x - middle) / step) + 8, 0, 15)
// with r16 the rounding to the cache's 16-bit type: codes are made against the pair that is stored.  (hi f - lo f and not
// (hi - lo) f: the range of a bfloat16 row may not fit a float32.)  step 0: code 8, the middle itself.  A group that holds a NaN
// or an infinity gets a NaN for both, as such an element would poison its row of a 16-bit cache.  Every operation is a single
// float32 one, rounded on its own: the codes of a key follow from the definition alone.  (lo + 8 step is one fused operation: 8 step is exact, but
// for the largest bfloat16 values it is beyond float32.)
//
// The reference keeps F32 and F16 caches only (crates/core-types/src/cache.rs); this format is this framework's own.
#include "packed_cache.cuh"

namespace {

template <typename T>
__device__ __forceinline__ float r16(float v) { return to_f32<T>(from_f32<T>(v)); }

template <typename T, int N> struct Elements { T v[N]; };

// One warp per (token, head slot); slots are Hq query heads, Hkv key heads, Hkv value heads.  Lane l owns elements l*E .. l*E + E - 1.  WIDE:
// it reads them, and those that they are turned with, in one piece (rows and halves aligned to E elements).
template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(256)
packed_write_kernel(const T* __restrict__ qkv, int ld, T* __restrict__ q_out, int ldq, const int* __restrict__ positions,
                    const int* __restrict__ req_of_token, const int* __restrict__ block_table, int table_width,
                    const float* __restrict__ cos_sin, int n_pos, uint8_t* __restrict__ plane, long long page_stride, int n_pages,
                    int page_size, int Hq, int Hkv, int R, int pairing, int write_kv, int* __restrict__ err) {
  constexpr int E = D / 32;
  using B = PackedBlock<D>;
  using Piece = Elements<T, E>;
  pdl_wait();
  pdl_launch();
  const int slots = Hq + (write_kv ? 2 * Hkv : 0);
  const int t = blockIdx.x, slot = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (slot >= slots) return;
  const T* src = qkv + (size_t)t * ld + (size_t)slot * D;
  float x[E];
  if (WIDE) {
    alignas(8) Piece p = *reinterpret_cast<const Piece*>(__builtin_assume_aligned(src + lane * E, 2 * E));
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32<T>(p.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32<T>(src[lane * E + e]);
  }
  const int pos = positions[t], half = R >> 1;
  if (pos < 0 || (half > 0 && pos >= n_pos)) {
    if (lane == 0) atomicExch(err, 2);
    return;
  }
  if (slot < Hq + Hkv && half > 0) {
    const float2* cs = reinterpret_cast<const float2*>(cos_sin) + (size_t)pos * half;
    float y[E], other[E];
    const int d0 = lane * E;
    if (pairing == 0) {
#pragma unroll
      for (int e = 0; e < E; ++e) other[e] = x[e ^ 1];
    } else if (WIDE) {
      alignas(8) Piece p = *reinterpret_cast<const Piece*>(__builtin_assume_aligned(src + (d0 < half ? d0 + half : d0 < R ? d0 - half : d0), 2 * E));
#pragma unroll
      for (int e = 0; e < E; ++e) other[e] = to_f32<T>(p.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = d0 + e;
        other[e] = to_f32<T>(src[d < half ? d + half : d < R ? d - half : d]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = d0 + e;
      y[e] = x[e];
      if (d < R) {
        const bool first = pairing == 0 ? (d & 1) == 0 : d < half;
        const float2 c = cs[pairing == 0 ? d >> 1 : (first ? d : d - half)];
        y[e] = first ? __fsub_rn(__fmul_rn(x[e], c.x), __fmul_rn(other[e], c.y)) : __fadd_rn(__fmul_rn(other[e], c.y), __fmul_rn(x[e], c.x));
      }
    }
    __syncwarp();      // q_out may be the row that the other lanes just read
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = y[e];
  }
  if (slot < Hq) {
    T* dst = q_out + (size_t)t * ldq + (size_t)slot * D + lane * E;
    if (WIDE) {
      alignas(8) Piece p;
#pragma unroll
      for (int e = 0; e < E; ++e) p.v[e] = from_f32<T>(x[e]);
      *reinterpret_cast<Piece*>(__builtin_assume_aligned(dst, 2 * E)) = p;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(x[e]);
    }
    return;
  }
  const int lp = pos / page_size;
  if (lp >= table_width) {
    if (lane == 0) atomicExch(err, 3);
    return;
  }
  const int page = block_table[(size_t)req_of_token[t] * table_width + lp];
  if (page < 0 || page >= n_pages) {
    if (lane == 0) atomicExch(err, 4);
    return;
  }
  const bool value = slot >= Hq + Hkv;
  const int h = slot - Hq - (value ? Hkv : 0);
  float lo = x[0], hi = x[0];
  bool wrong = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    wrong |= !isfinite(x[e]);
  }
#pragma unroll
  for (int o = PACKED_GROUP / E / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    wrong |= (bool)__shfl_xor_sync(0xffffffffu, (int)wrong, o);
  }
  float step = r16<T>(__fsub_rn(__fmul_rn(hi, 1.f / 15.f), __fmul_rn(lo, 1.f / 15.f)));
  float middle = r16<T>(fmaf(8.f, step, lo));
  if (wrong) step = middle = __int_as_float(0x7fc00000);
  unsigned codes = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float c = step > 0.f ? fminf(fmaxf(__fadd_rn(rintf(__fdiv_rn(__fsub_rn(x[e], middle), step)), 8.f), 0.f), 15.f) : 8.f;
    codes |= (unsigned)c << (4 * e);
  }
  const int in_page = pos % page_size, row = in_page % PACKED_POS;
  uint8_t* block = plane + (size_t)page * page_stride + ((size_t)h * (page_size / PACKED_POS) + in_page / PACKED_POS) * B::BYTES;
  uint8_t* dst = block + (value ? B::V_CODES : 0) + row * B::ROW + lane * (E / 2);
  if (E == 4) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)codes;
  else *dst = (uint8_t)codes;
  constexpr int LANES = PACKED_GROUP / E;      // lanes of a group
  if (lane % LANES == 0)
    reinterpret_cast<uint32_t*>(block + (value ? B::V_PAIRS : B::K_PAIRS))[row * B::GROUPS + lane / LANES] = pack2<T>(step, middle);
}

// The largest finite value of a 16-bit type: the rounding of a step may carry the outermost levels of a group beyond it.
template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return __uint_as_float(0x7f7f0000u); }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }

// One block per (item, KV head); a thread brings eight elements back: a word of codes in, 16 bytes out.
template <typename T, int D>
__global__ void __launch_bounds__(256)
unpack_kernel(const uint8_t* __restrict__ plane, long long page_stride, int n_pages, int page_size, const int* __restrict__ block_table,
              int table_width, const int* __restrict__ items, T* __restrict__ out, int Hkv, int* __restrict__ err) {
  using B = PackedBlock<D>;
  pdl_wait();
  pdl_launch();
  const int item = blockIdx.x, h = blockIdx.y;
  const int req = items[2 * item], lp = items[2 * item + 1];
  const int page = lp >= 0 && lp < table_width ? block_table[(size_t)req * table_width + lp] : -1;
  const bool missing = page < 0 || page >= n_pages;
  if (missing && threadIdx.x == 0) atomicExch(err, 5);
  const uint8_t* head = plane + (size_t)(missing ? 0 : page) * page_stride + (size_t)h * (page_size / PACKED_POS) * B::BYTES;
  constexpr int WORDS = D / 8;
  for (int i = threadIdx.x; i < 2 * page_size * WORDS; i += blockDim.x) {
    const int part = i / (page_size * WORDS), pos = i / WORDS % page_size, w = i % WORDS, row = pos % PACKED_POS;
    uint4 r = make_uint4(0, 0, 0, 0);
    if (!missing) {
      const uint8_t* block = head + (size_t)(pos / PACKED_POS) * B::BYTES;
      const unsigned codes = *reinterpret_cast<const unsigned*>(block + part * B::V_CODES + row * B::ROW + 4 * w);
      const unsigned pair = reinterpret_cast<const unsigned*>(block + (part ? B::V_PAIRS : B::K_PAIRS))[row * B::GROUPS + w * 8 / PACKED_GROUP];
      const float step = to_f32<T>(reinterpret_cast<const T*>(&pair)[0]), middle = to_f32<T>(reinterpret_cast<const T*>(&pair)[1]);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = fmaf(step, (float)((int)(codes >> (4 * k) & 15) - 8), middle);
        v[k] = x > largest<T>() ? largest<T>() : x < -largest<T>() ? -largest<T>() : x;      // (a NaN stays one)
      }
      r = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
    *reinterpret_cast<uint4*>(out + (((size_t)item * 2 + part) * Hkv + h) * page_size * D + (size_t)pos * D + w * 8) = r;
  }
}

}  // namespace

FERRUM_API int ferrum_packed_block_bytes(int D) { return D == 64 ? PackedBlock<64>::BYTES : D == 128 ? PackedBlock<128>::BYTES : 0; }

// qkv: [n_tokens, ld] rows of (q | k | v); q_out: [n_tokens, ldq], may be qkv itself.
FERRUM_API int ferrum_rope_cache_write_packed(const void* qkv, int dtype, int n_tokens, int ld, void* q_out, int ldq, const int* positions,
                                              const int* req_of_token, const int* block_table, int table_width, const float* cos_sin,
                                              int n_pos, void* plane, long long page_stride, int n_pages, int page_size, int Hq, int Hkv,
                                              int D, int R, int pairing, int write_kv, int* err_flag, cudaStream_t stream) {
  FERRUM_CHECK_ARG(n_tokens >= 0 && Hq > 0 && Hkv > 0, "rope_packed: bad sizes T=%d Hq=%d Hkv=%d", n_tokens, Hq, Hkv);
  FERRUM_CHECK_ARG(D == 64 || D == 128, "rope_packed: a cache in 4 bits has heads of 64 or 128 elements, found %d", D);
  FERRUM_CHECK_ARG(R >= 0 && R % 2 == 0 && R <= D, "rope_packed: rope_dim %d must be even and at most head_dim %d", R, D);
  FERRUM_CHECK_ARG(ld >= (Hq + 2 * Hkv) * D && ldq >= Hq * D, "rope_packed: rows of %d and %d elements are too short", ld, ldq);
  FERRUM_CHECK_ARG(pairing == 0 || pairing == 1, "rope_packed: pairing code %d", pairing);
  FERRUM_CHECK_ARG(!write_kv || (packed_page_ok(page_size) && table_width > 0 && plane && n_pages > 0),
                   "rope_packed: page size %d must be a multiple of %d, and the cache given", page_size, PACKED_POS);
  FERRUM_CHECK_ARG(((uintptr_t)plane & 15) == 0 && page_stride % 16 == 0, "rope_packed: pages must be 16-byte aligned");
  if (n_tokens == 0) return 0;
  const int slots = Hq + (write_kv ? 2 * Hkv : 0), E = D / 32;
  const dim3 grid(n_tokens, (slots + 7) / 8);
  FERRUM_CHECK_ARG(grid.y <= 65535, "rope_packed: too many heads");
  const bool wide = ld % E == 0 && ldq % E == 0 && (((uintptr_t)qkv | (uintptr_t)q_out) & (2 * E - 1)) == 0 && (pairing == 0 || R / 2 % E == 0);
  auto launch = [&](auto kernel, auto* x, auto* q) {
    launch_kernel(kernel, grid, dim3(256), 0, stream, x, ld, q, ldq, positions, req_of_token, block_table, table_width, cos_sin, n_pos, (uint8_t*)plane,
                  page_stride, n_pages, page_size, Hq, Hkv, R, pairing, write_kv, err_flag);
  };
  FERRUM_DISPATCH_16BIT(dtype, T, {
    if (D == 64) wide ? launch(packed_write_kernel<T, 64, true>, (const T*)qkv, (T*)q_out) : launch(packed_write_kernel<T, 64, false>, (const T*)qkv, (T*)q_out);
    else wide ? launch(packed_write_kernel<T, 128, true>, (const T*)qkv, (T*)q_out) : launch(packed_write_kernel<T, 128, false>, (const T*)qkv, (T*)q_out);
  });
  FERRUM_CHECK_LAUNCH("rope_cache_write_packed");
  return 0;
}

// items: [n_items][2] int32 (request, page of the request); out: [n_items][2][Hkv][page_size][D].
FERRUM_API int ferrum_unpack_cache(const void* plane, long long page_stride, int n_pages, int page_size, const int* block_table, int table_width,
                                   const int* items, int n_items, void* out, int dtype, int Hkv, int D, int* err_flag, cudaStream_t stream) {
  FERRUM_CHECK_ARG(D == 64 || D == 128, "unpack_cache: a cache in 4 bits has heads of 64 or 128 elements, found %d", D);
  FERRUM_CHECK_ARG(packed_page_ok(page_size) && table_width > 0 && n_pages > 0 && Hkv > 0 && Hkv <= 65535 && n_items >= 0,
                   "unpack_cache: bad sizes (page size %d must be a multiple of %d)", page_size, PACKED_POS);
  FERRUM_CHECK_ARG((((uintptr_t)plane | (uintptr_t)out) & 15) == 0 && page_stride % 16 == 0, "unpack_cache: operands must be 16-byte aligned");
  if (n_items == 0) return 0;
  const dim3 grid(n_items, Hkv);
  FERRUM_DISPATCH_16BIT(dtype, T, {
    if (D == 64) launch_kernel(unpack_kernel<T, 64>, grid, dim3(256), 0, stream, (const uint8_t*)plane, page_stride, n_pages, page_size, block_table, table_width, items, (T*)out, Hkv, err_flag);
    else launch_kernel(unpack_kernel<T, 128>, grid, dim3(256), 0, stream, (const uint8_t*)plane, page_stride, n_pages, page_size, block_table, table_width, items, (T*)out, Hkv, err_flag);
  });
  FERRUM_CHECK_LAUNCH("unpack_cache");
  return 0;
}
