// Causal grouped-query attention of decoded tokens over a cache held in 4 bits (packed_cache.cuh has the layout):
//   o = sum_j p_j v_j,  p = softmax_j(scale * q . k_j),  over the keys j of the request up to the token itself, the last `window` of them
// where a window is set.
//
// Simplest form: a block per (request, KV head) walks its rows one after the other; its four warps take every fourth key, a lane holds
// D / 32 elements, the softmax runs with the data, and the warps' (maximum, sum, values) meet at the end.
#include "packed_cache.cuh"

namespace {

struct PackedParams {
  const void* q;
  void* out;
  const uint8_t* plane;
  const int* block_table;
  const int* q_start;
  const int* pos0;
  int* err;
  long long page_stride;
  int ldq, ldo, n_pages, page_size, table_width, Hq, Hkv, window;
  float scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(128)
attention_packed_kernel(const PackedParams p) {
  using B = PackedBlock<D>;
  constexpr int E = D / 32;
  __shared__ float s_ml[4][2], s_o[4][D];
  pdl_launch();
  pdl_wait();
  const int req = blockIdx.x, kvh = blockIdx.y, G = p.Hq / p.Hkv;
  const int qs = p.q_start[req], n = p.q_start[req + 1] - qs;
  if (n * G > PACKED_FEW_ROWS) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pos0 = p.pos0[req];
  for (int r = 0; r < n * G; ++r) {
    const int token = qs + r / G, head = kvh * G + r % G, at = pos0 + r / G;
    const T* q = (const T*)p.q + (size_t)token * p.ldq + (size_t)head * D + lane * E;
    float x[E], o[E], m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; ++e) x[e] = to_f32<T>(q[e]) * p.scale, o[e] = 0.f;
    for (int key = max(0, p.window > 0 ? at - p.window + 1 : 0) + warp; key <= at; key += 4) {
      const int lp = key / p.page_size, in_page = key % p.page_size, row = in_page % PACKED_POS;
      const int page = lp < p.table_width ? p.block_table[(size_t)req * p.table_width + lp] : -1;
      if (page < 0 || page >= p.n_pages) {
        if (lane == 0) atomicExch(p.err, 5);
        continue;
      }
      const uint8_t* block = p.plane + (size_t)page * p.page_stride + ((size_t)kvh * (p.page_size / PACKED_POS) + in_page / PACKED_POS) * B::BYTES;
      const T* kp = (const T*)(block + B::K_PAIRS) + (row * B::GROUPS + lane * E / PACKED_GROUP) * 2;
      const T* vp = (const T*)(block + B::V_PAIRS) + (row * B::GROUPS + lane * E / PACKED_GROUP) * 2;
      const uint8_t* kc = block + row * B::ROW + lane * (E / 2);
      float dot = 0.f;
      for (int e = 0; e < E; ++e) dot += x[e] * (to_f32<T>(kp[1]) + to_f32<T>(kp[0]) * (float)((kc[e / 2] >> (4 * (e & 1)) & 15) - 8));
      dot = warp_sum(dot);
      const float m_new = fmaxf(m, dot), keep = m == -INFINITY ? 0.f : expf(m - m_new), w = expf(dot - m_new);
      l = l * keep + w;
      for (int e = 0; e < E; ++e)
        o[e] = o[e] * keep + w * (to_f32<T>(vp[1]) + to_f32<T>(vp[0]) * (float)((kc[B::V_CODES + e / 2] >> (4 * (e & 1)) & 15) - 8));
      m = m_new;
    }
    if (lane == 0) s_ml[warp][0] = m, s_ml[warp][1] = l;
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    __syncthreads();
    if (warp == 0) {
      float M = -INFINITY, L = 0.f, acc[E] = {};
      for (int w = 0; w < 4; ++w) M = fmaxf(M, s_ml[w][0]);
      for (int w = 0; w < 4; ++w) {
        const float f = s_ml[w][0] == -INFINITY ? 0.f : expf(s_ml[w][0] - M);
        L += s_ml[w][1] * f;
        for (int e = 0; e < E; ++e) acc[e] += s_o[w][lane * E + e] * f;
      }
      for (int e = 0; e < E; ++e) ((T*)p.out)[(size_t)token * p.ldo + (size_t)head * D + lane * E + e] = from_f32<T>(L > 0.f ? acc[e] / L : 0.f);
    }
    __syncthreads();
  }
}

}  // namespace

FERRUM_API int ferrum_attention_packed_rows() { return PACKED_FEW_ROWS; }

// Floats of workspace that a call needs.
FERRUM_API long long ferrum_attention_packed_workspace(int D) { return 0; }

FERRUM_API int ferrum_attention_packed(const void* q, int ldq, void* out, int ldo, int dtype, const void* plane, long long page_stride, int n_pages,
                                       int page_size, const int* block_table, int table_width, const int* q_start, const int* pos0, int n_reqs,
                                       int n_tokens, float* part, long long part_floats, int Hq, int Hkv, int D, float scale, int window,
                                       int* err_flag, cudaStream_t stream) {
  FERRUM_CHECK_ARG(Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "attention_packed: bad head counts Hq=%d Hkv=%d", Hq, Hkv);
  FERRUM_CHECK_ARG(D == 64 || D == 128, "attention_packed: a cache in 4 bits has heads of 64 or 128 elements, found %d", D);
  FERRUM_CHECK_ARG(packed_page_ok(page_size) && table_width > 0 && n_pages > 0 && window >= 0 && n_reqs >= 0 && n_tokens >= 0,
                   "attention_packed: bad sizes (page size %d must be a multiple of %d)", page_size, PACKED_POS);
  FERRUM_CHECK_ARG(err_flag != nullptr, "attention_packed: the error flag is required");
  FERRUM_CHECK_ARG((((uintptr_t)q | (uintptr_t)out | (uintptr_t)plane) & 15) == 0 && ldq % 8 == 0 && ldo % 8 == 0 && page_stride % 16 == 0,
                   "attention_packed: operands must be 16-byte aligned");
  FERRUM_CHECK_ARG(ldq >= Hq * D && ldo >= Hq * D, "attention_packed: rows of %d and %d elements are too short", ldq, ldo);
  FERRUM_CHECK_ARG(part_floats >= ferrum_attention_packed_workspace(D), "attention_packed: the workspace is too small");
  if (n_reqs == 0 || n_tokens == 0) return 0;
  PackedParams p{q, out, (const uint8_t*)plane, block_table, q_start, pos0, err_flag, page_stride, ldq, ldo, n_pages, page_size, table_width, Hq, Hkv, window, scale};
  FERRUM_DISPATCH_16BIT(dtype, T, {
    if (D == 64) launch_kernel(attention_packed_kernel<T, 64>, dim3(n_reqs, Hkv), dim3(128), 0, stream, p);
    else launch_kernel(attention_packed_kernel<T, 128>, dim3(n_reqs, Hkv), dim3(128), 0, stream, p);
  });
  FERRUM_CHECK_LAUNCH("attention_packed");
  return 0;
}
