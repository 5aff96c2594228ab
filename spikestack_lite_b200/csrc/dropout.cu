// Dropout from a counter-based generator, with the residual added:
//   Y[i] = R[i] + (w_i >= round(p 2^32) ? X[i] / (1 - p) : 0)
// where w_i is word i % 4 of Philox4x32 with 7 rounds (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011; 7 rounds are
// the fewest the paper found to pass every test of its battery) at counter
// (i / 4, offset) under the key `seed`.  The mask is a function of (seed,
// offset, i): it is never stored, and the backward pass is the same kernel on
// the output's gradient without a residual.
//
// Bound: HBM for fp32 (2 or 3 tensors moved once); for 16-bit elements the
// generator's integer multiplies come close to it (14 32x32->64 products per
// four elements), which is why it runs 7 rounds and not 10.  Measured on
// 262144x512 bf16: 133 us with the residual (92 % of the time its bytes need at
// the measured HBM rate), 100 us without (82 %, the generator).
#include "elem.cuh"

namespace spk {

struct DropoutArgs {
  const void* x;
  const void* r;          // or null
  void* y;
  int64_t n;
  uint64_t seed, offset;  // used when key is null
  const int64_t* key;     // (seed, offset) on the device, or null
  uint32_t threshold;     // kept where word >= threshold
  float scale;
};

struct Philox7 {
  uint32_t k0[7], k1[7], o0, o1;  // the rounds' keys, the counter's upper half

  __device__ __forceinline__ Philox7(uint64_t seed, uint64_t offset) : o0((uint32_t)offset), o1((uint32_t)(offset >> 32)) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      k0[r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
      k1[r] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
    }
  }

  __device__ __forceinline__ uint4 operator()(uint64_t counter) const {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = o0, c3 = o1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      const uint64_t m0 = (uint64_t)c0 * 0xD2511F53u, m1 = (uint64_t)c2 * 0xCD9E8D57u;
      const uint32_t n0 = (uint32_t)(m1 >> 32) ^ c1 ^ k0[r];
      const uint32_t n2 = (uint32_t)(m0 >> 32) ^ c3 ^ k1[r];
      c1 = (uint32_t)m1;
      c3 = (uint32_t)m0;
      c0 = n0;
      c2 = n2;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

constexpr int kDropThreads = 256;

template <typename E, bool RES, int V>
__device__ __forceinline__ Pack<E, V> dropout_pack(const Pack<E, V>& x, const Pack<E, V>& r, const Philox7& rng,
                                                   int64_t i, uint32_t threshold, float scale) {
  float y[V];
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const uint4 w = rng((uint64_t)(i * (V / 4) + q));
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // a dropped element contributes 0 whatever it holds (no inf * 0)
      const float v = ws[j] >= threshold ? elem_to_f32(x.e[4 * q + j]) : 0.0f;
      y[4 * q + j] = RES ? fmaf(v, scale, elem_to_f32(r.e[4 * q + j])) : v * scale;
    }
  }
  return pack_f32<E, V>(y);
}

// A thread takes U packs of V = 4 or 8 consecutive elements (16 bytes, V / 4
// counters) at a time.  ALIGNED: every tensor is 16-byte aligned and the
// accesses are 16 bytes wide; otherwise they are single elements, of the same
// counters.  The last, partial pack goes by elements too.  Once every thread of
// a full GPU has a pack, U = 2 with a residual and 4 without (262144x512 bf16,
// us: 155, 133 and 139 with one, two and four packs in flight; without a
// residual 156, 106 and 100); below that 1, to spread few packs.
template <typename E, bool RES, bool ALIGNED, int U>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(DropoutArgs a) {
  constexpr int V = 16 / (int)sizeof(E);
  const uint64_t seed = a.key != nullptr ? (uint64_t)a.key[0] : a.seed;
  const uint64_t offset = a.key != nullptr ? (uint64_t)a.key[1] : a.offset;
  const Philox7 rng(seed, offset);
  const E* const X = static_cast<const E*>(a.x);
  const E* const R = static_cast<const E*>(a.r);
  E* const Y = static_cast<E*>(a.y);
  const int64_t whole = ALIGNED ? a.n / V : 0;
  const int64_t step = (int64_t)gridDim.x * kDropThreads * U;
  for (int64_t i0 = (int64_t)blockIdx.x * kDropThreads * U + threadIdx.x; i0 < whole; i0 += step) {
    Pack<E, V> x[U], r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * kDropThreads;
      if (i < whole) {
        x[u] = load_pack<E, V>(X + i * V);
        if (RES) r[u] = load_pack<E, V>(R + i * V);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * kDropThreads;
      if (i < whole) store_pack<E, V>(Y + i * V, dropout_pack<E, RES, V>(x[u], r[u], rng, i, a.threshold, a.scale));
    }
  }
  const int64_t vecs = ceil_div(a.n, V);
  for (int64_t i = whole + (int64_t)blockIdx.x * kDropThreads + threadIdx.x; i < vecs;
       i += (int64_t)gridDim.x * kDropThreads) {
    Pack<E, V> x, r;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = i * V + j < a.n;
      x.e[j] = in ? X[i * V + j] : elem_from_f32<E>(0.0f);
      r.e[j] = RES && in ? R[i * V + j] : elem_from_f32<E>(0.0f);
    }
    const Pack<E, V> y = dropout_pack<E, RES, V>(x, r, rng, i, a.threshold, a.scale);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i * V + j < a.n) Y[i * V + j] = y.e[j];
  }
}

template <typename E, bool RES>
static void dropout_launch(const DropoutArgs& a, bool aligned, cudaStream_t st) {
  const int64_t vecs = ceil_div(a.n, (int64_t)(16 / sizeof(E))), most = (int64_t)sm_count() * 8;
  const unsigned blocks = (unsigned)min64(ceil_div(vecs, kDropThreads), most);
  if (!aligned)
    dropout_kernel<E, RES, false, 1><<<blocks, kDropThreads, 0, st>>>(a);
  else if (vecs <= most * kDropThreads)
    dropout_kernel<E, RES, true, 1><<<blocks, kDropThreads, 0, st>>>(a);
  else
    dropout_kernel<E, RES, true, RES ? 2 : 4><<<blocks, kDropThreads, 0, st>>>(a);
}

}  // namespace spk

extern "C" int spk_dropout(const void* X, const void* R, int dtype, int64_t n, double p, uint64_t seed,
                           uint64_t offset, const int64_t* key, void* Y, spk_stream_t stream) {
  SPK_REQUIRE(n >= 0, "invalid element count (n=%lld)", (long long)n);
  SPK_REQUIRE(p >= 0.0 && p <= 1.0, "p must lie in [0, 1]");
  const size_t eb = spk::elem_bytes(dtype);
  SPK_REQUIRE(eb != 0, "unknown element type %d", dtype);
  if (n == 0) return SPK_OK;
  SPK_REQUIRE(X != nullptr && Y != nullptr, "X and Y must be non-null");
  SPK_REQUIRE(spk::aligned_to(X, eb) && spk::aligned_to(R, eb) && spk::aligned_to(Y, eb) && spk::aligned_to(key, 8),
              "tensors must be aligned to their elements");
  cudaStream_t st = (cudaStream_t)stream;
  const uint64_t threshold = (uint64_t)(p * 4294967296.0 + 0.5);
  if (threshold > 0xffffffffull) {  // nothing is kept
    if (R == nullptr)
      SPK_CUDA_TRY(cudaMemsetAsync(Y, 0, (size_t)n * eb, st));
    else if (Y != R)
      SPK_CUDA_TRY(cudaMemcpyAsync(Y, R, (size_t)n * eb, cudaMemcpyDeviceToDevice, st));
    return SPK_OK;
  }
  spk::DropoutArgs a{};
  a.x = X;
  a.r = R;
  a.y = Y;
  a.n = n;
  a.seed = seed;
  a.offset = offset;
  a.key = key;
  a.threshold = (uint32_t)threshold;
  a.scale = (float)(1.0 / (1.0 - p));
  const bool aligned = spk::aligned_to(X, 16) && spk::aligned_to(R, 16) && spk::aligned_to(Y, 16);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    if (R != nullptr)
      spk::dropout_launch<E, true>(a, aligned, st);
    else
      spk::dropout_launch<E, false>(a, aligned, st);
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
  return SPK_OK;
}
