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
// Both kernels move bytes: the write reads a token's row and writes 9 D / 8 bytes a KV head (2,048 tokens of 48 head slots of 128 and their cosines, 45 MB: 21 us
// from DRAM, 2.2 TB/s, 15 from the L2; a few tokens take the 4 us of a launch and of one chain of loads, shuffles and divisions); the unpacking writes 3.6 times what it reads (2,048
// positions, 8 KV heads of 128, 10.7 MB: 5.7 us; 10,208 of them, 53 MB: 14 us, 3.8 TB/s).
//
// The reference keeps F32 and F16 caches only (crates/core-types/src/cache.rs); this format is this framework's own.
#include "packed_cache.cuh"

namespace {

template <typename T>
__device__ __forceinline__ float r16(float v) { return to_f32<T>(from_f32<T>(v)); }

// Eight warps a token; warp w of blockIdx.y's share does head slots first + w, first + w + 8, ... (SLOTS of them): Hq query heads, Hkv key
// heads, Hkv value heads.  Lane l owns elements l*E .. l*E + E - 1 of a head and keeps their cosines and sines for all of its heads.  WIDE:
// rows and halves are aligned to E elements, so that a lane reads its own in one piece and has those they are turned with from another lane.
// Few tokens: a slot a warp, so that a token's heads are written at once.  Many: six, since the cosines and sines are four times a
// head's bytes (B200, 48 slots of 128, one / six: 2,048 tokens 29 / 21 us; 290 tokens,
// with the pages brought back, 7.9 / 6.1, 150 tokens 5.7 / 5.8).
template <typename T, int D, bool WIDE, int SLOTS>
__global__ void __launch_bounds__(256)
packed_write_kernel(const T* __restrict__ qkv, int ld, T* __restrict__ q_out, int ldq, const int* __restrict__ positions,
                    const int* __restrict__ req_of_token, const int* __restrict__ block_table, int table_width,
                    const float* __restrict__ cos_sin, int n_pos, uint8_t* __restrict__ plane, long long page_stride, int n_pages,
                    int page_size, int Hq, int Hkv, int R, int pairing, int write_kv, int* __restrict__ err) {
  constexpr int E = D / 32, W = E / 2;
  using B = PackedBlock<D>;
  pdl_wait();
  pdl_launch();
  const int slots = Hq + (write_kv ? 2 * Hkv : 0);
  const int t = blockIdx.x, slot0 = blockIdx.y * 8 * SLOTS + (threadIdx.x >> 5), lane = threadIdx.x & 31, d0 = lane * E;
  const T* row = qkv + (size_t)t * ld;
  if (slot0 >= slots) return;
  uint32_t raw[SLOTS][W];
  if (WIDE) {
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
      if (slot0 + 8 * i < slots) {
        const T* src = row + (size_t)(slot0 + 8 * i) * D + d0;
        if (W == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(src);
          raw[i][0] = v.x;
          raw[i][W - 1] = v.y;
        } else {
          raw[i][0] = *reinterpret_cast<const uint32_t*>(src);
        }
      }
  }
  const int pos = positions[t], half = R >> 1;
  if (pos < 0 || (half > 0 && pos >= n_pos)) {
    if (lane == 0) atomicExch(err, 2);
    return;
  }
  float2 cs[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = d0 + e;
    cs[e] = d < R ? reinterpret_cast<const float2*>(cos_sin)[(size_t)pos * half + (pairing == 0 ? d >> 1 : d < half ? d : d - half)] : make_float2(1.f, 0.f);
  }
  uint8_t* page_at = nullptr;
  const int in_page = pos % page_size, block_row = in_page % PACKED_POS;
  if (write_kv && slot0 + 8 * (SLOTS - 1) >= Hq) {
    const int lp = pos / page_size;
    if (lp >= table_width) {
      if (lane == 0) atomicExch(err, 3);
    } else {
      const int page = block_table[(size_t)req_of_token[t] * table_width + lp];
      if (page < 0 || page >= n_pages) {
        if (lane == 0) atomicExch(err, 4);
      } else {
        page_at = plane + (size_t)page * page_stride + (size_t)(in_page / PACKED_POS) * B::BYTES;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int slot = slot0 + 8 * i;
    if (slot >= slots) break;
    const T* src = row + (size_t)slot * D;
    float x[E];
    if (WIDE) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const T* v = reinterpret_cast<const T*>(&raw[i][w]);
        x[2 * w] = to_f32<T>(v[0]);
        x[2 * w + 1] = to_f32<T>(v[1]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = to_f32<T>(src[d0 + e]);
    }
    if (slot < Hq + Hkv && half > 0) {
      float other[E];
      if (pairing == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) other[e] = x[e ^ 1];
      } else if (WIDE) {
        const int from = d0 < half ? lane + half / E : d0 < R ? lane - half / E : lane;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t o = __shfl_sync(0xffffffffu, raw[i][w], from);
          const T* v = reinterpret_cast<const T*>(&o);
          other[2 * w] = to_f32<T>(v[0]);
          other[2 * w + 1] = to_f32<T>(v[1]);
        }
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
        const bool first = pairing == 0 ? (d & 1) == 0 : d < half;
        const float y = first ? __fsub_rn(__fmul_rn(x[e], cs[e].x), __fmul_rn(other[e], cs[e].y)) : __fadd_rn(__fmul_rn(other[e], cs[e].y), __fmul_rn(x[e], cs[e].x));
        if (d < R) x[e] = y;
      }
      __syncwarp();      // q_out may be the row that the other lanes just read
    }
    if (slot < Hq) {
      T* dst = q_out + (size_t)t * ldq + (size_t)slot * D + d0;
      if (WIDE && W == 2) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[E - 2], x[E - 1]));
      } else if (WIDE) {
        *reinterpret_cast<uint32_t*>(dst) = pack2<T>(x[0], x[1]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(x[e]);
      }
      continue;
    }
    if (page_at == nullptr) continue;
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
    }
    const unsigned bad = __ballot_sync(0xffffffffu, wrong);
    constexpr int LANES = PACKED_GROUP / E;      // lanes of a group
    const unsigned of_group = (LANES == 32 ? 0xffffffffu : (1u << (LANES % 32)) - 1) << (lane / LANES * (LANES % 32));
    float step = r16<T>(__fsub_rn(__fmul_rn(hi, 1.f / 15.f), __fmul_rn(lo, 1.f / 15.f)));
    float middle = r16<T>(fmaf(8.f, step, lo));
    if (bad & of_group) step = middle = __int_as_float(0x7fc00000);
    // the quotient by a reciprocal is off by three roundings: it names the same whole number as the quotient itself unless it is next to a half, and
    // there, or where the reciprocal is no number, the division decides
    unsigned codes = 0;
    const float inverse = __frcp_rn(step);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = __fsub_rn(x[e], middle), q = __fmul_rn(d, inverse);
      float c = rintf(q);
      if (!(fabsf(q - c) < 0.4999f)) c = rintf(__fdiv_rn(d, step));
      c = step > 0.f ? fminf(fmaxf(__fadd_rn(c, 8.f), 0.f), 15.f) : 8.f;
      codes |= (unsigned)c << (4 * e);
    }
    uint8_t* block = page_at + (size_t)h * (page_size / PACKED_POS) * B::BYTES;
    uint8_t* dst = block + (value ? B::V_CODES : 0) + block_row * B::ROW + lane * (E / 2);
    if (E == 4) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)codes;
    else *dst = (uint8_t)codes;
    if (lane % LANES == 0)
      reinterpret_cast<uint32_t*>(block + (value ? B::V_PAIRS : B::K_PAIRS))[block_row * B::GROUPS + lane / LANES] = pack2<T>(step, middle);
  }
}

// The largest finite value of a 16-bit type: the rounding of a step may carry the outermost levels of a group beyond it.
template <typename T> __device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<__nv_bfloat16>() { return __uint_as_float(0x7f7f0000u); }
template <> __device__ __forceinline__ float largest<__half>() { return 65504.f; }

// One block per (item, KV head); a thread brings eight elements back at a time: a word of codes in, 16 bytes out, both of its rows of a block of
// 16 positions (and of keys and values) on their way together.
// middle + (code - 8) step is rounded to the 16-bit type, since that is what the kernels of prompt portions read: an output's error against 64 bits
// becomes that of a 16-bit cache, 0.003 to 0.004 in bfloat16 and 0.0004 in float16 (0.0017 and 0.0002 for rounding the result alone).
// 32-bit pages would want kernels of their own and twice the bytes written.
template <typename T, int D>
__global__ void __launch_bounds__(256)
unpack_kernel(const uint8_t* __restrict__ plane, long long page_stride, int n_pages, int page_size, const int* __restrict__ block_table,
              int table_rows, int table_width, const int* __restrict__ items, T* __restrict__ out, int Hkv, int* __restrict__ err) {
  using B = PackedBlock<D>;
  constexpr int WORDS = D / 8, AT_ONCE = 256 / WORDS, ROUNDS = (2 * PACKED_POS + AT_ONCE - 1) / AT_ONCE;      // rows of keys and values of a block
  pdl_wait();
  pdl_launch();
  const int item = blockIdx.x, h = blockIdx.y;
  const int req = items[2 * item], lp = items[2 * item + 1];
  const int page = req >= 0 && req < table_rows && lp >= 0 && lp < table_width ? block_table[(size_t)req * table_width + lp] : -1;
  const bool missing = page < 0 || page >= n_pages;
  if (missing && threadIdx.x == 0) atomicExch(err, 5);
  const uint8_t* head = plane + (size_t)(missing ? 0 : page) * page_stride + (size_t)h * (page_size / PACKED_POS) * B::BYTES;
  T* dst = out + ((size_t)item * 2 * Hkv + h) * page_size * D;
  const size_t to_values = (size_t)Hkv * page_size * D;
  const int w = threadIdx.x % WORDS, first = threadIdx.x / WORDS;
#pragma unroll 2
  for (int block = 0; block < page_size / PACKED_POS; ++block, head += B::BYTES, dst += PACKED_POS * D) {
    unsigned codes[ROUNDS], pair[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int row = first + i * AT_ONCE, part = row / PACKED_POS, pos = row % PACKED_POS;
      codes[i] = pair[i] = 0;                       // (a missing page: step and middle 0)
      if (!missing) {
        codes[i] = *reinterpret_cast<const unsigned*>(head + part * B::V_CODES + pos * B::ROW + 4 * w);
        pair[i] = reinterpret_cast<const unsigned*>(head + (part ? B::V_PAIRS : B::K_PAIRS))[pos * B::GROUPS + w * 8 / PACKED_GROUP];
      }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int row = first + i * AT_ONCE, part = row / PACKED_POS, pos = row % PACKED_POS;
      const float step = to_f32<T>(reinterpret_cast<const T*>(&pair[i])[0]), middle = to_f32<T>(reinterpret_cast<const T*>(&pair[i])[1]);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)      // 2^23 + code by its bits, less 2^23 + 8
        v[k] = fmaf(step, __uint_as_float((codes[i] >> (4 * k) & 15u) | 0x4B000000u) - 8388616.f, middle);
      if (!(fabsf(middle) + 8.f * step < largest<T>())) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = v[k] > largest<T>() ? largest<T>() : v[k] < -largest<T>() ? -largest<T>() : v[k];      // (a NaN stays one)
      }
      *reinterpret_cast<uint4*>(dst + part * to_values + pos * D + w * 8) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
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
  FERRUM_CHECK_ARG(err_flag != nullptr, "rope_packed: the error flag is required");
  if (n_tokens == 0) return 0;
  const int slots = Hq + (write_kv ? 2 * Hkv : 0), E = D / 32;
  const bool wide = ld % E == 0 && ldq % E == 0 && (((uintptr_t)qkv | (uintptr_t)q_out) & (2 * E - 1)) == 0 && (pairing == 0 || R / 2 % E == 0);
  const int a_warp = wide && 2 * n_tokens >= 3 * ferrum_sm_count() ? 6 : 1;
  const dim3 grid(n_tokens, (slots + 8 * a_warp - 1) / (8 * a_warp));
  FERRUM_CHECK_ARG(grid.y <= 65535, "rope_packed: too many heads");
  auto launch = [&](auto kernel, auto* x, auto* q) {
    launch_kernel(kernel, grid, dim3(256), 0, stream, x, ld, q, ldq, positions, req_of_token, block_table, table_width, cos_sin, n_pos, (uint8_t*)plane,
                  page_stride, n_pages, write_kv ? page_size : PACKED_POS, Hq, Hkv, R, pairing, write_kv, err_flag);
  };
  FERRUM_DISPATCH_16BIT(dtype, T, {
    const T* x = (const T*)qkv;
    T* q = (T*)q_out;
    if (D == 64) {
      if (!wide) launch(packed_write_kernel<T, 64, false, 1>, x, q);
      else if (a_warp == 1) launch(packed_write_kernel<T, 64, true, 1>, x, q);
      else launch(packed_write_kernel<T, 64, true, 6>, x, q);
    } else {
      if (!wide) launch(packed_write_kernel<T, 128, false, 1>, x, q);
      else if (a_warp == 1) launch(packed_write_kernel<T, 128, true, 1>, x, q);
      else launch(packed_write_kernel<T, 128, true, 6>, x, q);
    }
  });
  FERRUM_CHECK_LAUNCH("rope_cache_write_packed");
  return 0;
}

// items: [n_items][2] int32 (request, page of the request); out: [n_items][2][Hkv][page_size][D].
FERRUM_API int ferrum_unpack_cache(const void* plane, long long page_stride, int n_pages, int page_size, const int* block_table, int table_rows, int table_width,
                                   const int* items, int n_items, void* out, int dtype, int Hkv, int D, int* err_flag, cudaStream_t stream) {
  FERRUM_CHECK_ARG(D == 64 || D == 128, "unpack_cache: a cache in 4 bits has heads of 64 or 128 elements, found %d", D);
  FERRUM_CHECK_ARG(packed_page_ok(page_size) && table_width > 0 && n_pages > 0 && Hkv > 0 && Hkv <= 65535 && n_items >= 0,
                   "unpack_cache: bad sizes (page size %d must be a multiple of %d)", page_size, PACKED_POS);
  FERRUM_CHECK_ARG((((uintptr_t)plane | (uintptr_t)out) & 15) == 0 && page_stride % 16 == 0, "unpack_cache: operands must be 16-byte aligned");
  FERRUM_CHECK_ARG(err_flag != nullptr, "unpack_cache: the error flag is required");
  if (n_items == 0) return 0;
  const dim3 grid(n_items, Hkv);
  FERRUM_DISPATCH_16BIT(dtype, T, {
    if (D == 64) launch_kernel(unpack_kernel<T, 64>, grid, dim3(256), 0, stream, (const uint8_t*)plane, page_stride, n_pages, page_size, block_table, table_rows, table_width, items, (T*)out, Hkv, err_flag);
    else launch_kernel(unpack_kernel<T, 128>, grid, dim3(256), 0, stream, (const uint8_t*)plane, page_stride, n_pages, page_size, block_table, table_rows, table_width, items, (T*)out, Hkv, err_flag);
  });
  FERRUM_CHECK_LAUNCH("unpack_cache");
  return 0;
}
