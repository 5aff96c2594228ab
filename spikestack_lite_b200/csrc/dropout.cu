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
// four elements), which is why it runs 7 rounds and not 10.
#include "elem.cuh"

namespace spk {

struct DropoutArgs {
  const void* x;
  const void* r;         // or null
  void* y;
  int64_t n;
  uint64_t seed, offset;  // used when key is null
  const int64_t* key;     // (seed, offset) on the device, or null
  uint64_t threshold;     // kept where word >= threshold (2^32: none)
  float scale;
};

struct Philox7 {
  uint32_t k0, k1, o0, o1;

  __device__ __forceinline__ Philox7(uint64_t seed, uint64_t offset)
      : k0((uint32_t)seed), k1((uint32_t)(seed >> 32)), o0((uint32_t)offset), o1((uint32_t)(offset >> 32)) {}

  __device__ __forceinline__ uint4 operator()(uint64_t counter) const {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = o0, c3 = o1;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
      const uint64_t m0 = (uint64_t)c0 * 0xD2511F53u, m1 = (uint64_t)c2 * 0xCD9E8D57u;
      const uint32_t n0 = (uint32_t)(m1 >> 32) ^ c1 ^ (k0 + (uint32_t)r * 0x9E3779B9u);
      const uint32_t n2 = (uint32_t)(m0 >> 32) ^ c3 ^ (k1 + (uint32_t)r * 0xBB67AE85u);
      c1 = (uint32_t)m1;
      c3 = (uint32_t)m0;
      c0 = n0;
      c2 = n2;
    }
    return make_uint4(c0, c1, c2, c3);
  }
};

// A thread takes V = 4 or 8 consecutive elements (16 bytes) at a time: V / 4
// counters.  ALIGNED: every tensor is 16-byte aligned and the accesses are
// 16 bytes wide; otherwise they are single elements, of the same counters.
template <typename E, bool ALIGNED>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a) {
  constexpr int V = 16 / (int)sizeof(E);
  const uint64_t seed = a.key != nullptr ? (uint64_t)a.key[0] : a.seed;
  const uint64_t offset = a.key != nullptr ? (uint64_t)a.key[1] : a.offset;
  const Philox7 rng(seed, offset);
  const E* X = static_cast<const E*>(a.x);
  const E* R = static_cast<const E*>(a.r);
  E* Y = static_cast<E*>(a.y);
  const bool none = a.threshold > 0xffffffffull;
  const uint32_t thr = (uint32_t)a.threshold;
  const int64_t vecs = ceil_div(a.n, V), step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < vecs; i += step) {
    const int64_t at = i * V;
    const bool whole = at + V <= a.n;
    Pack<E, V> x, r, y;
    if (ALIGNED && whole) {
      x = load_pack<E, V>(X + at);
      if (R != nullptr) r = load_pack<E, V>(R + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (at + j < a.n) {
          x.e[j] = X[at + j];
          if (R != nullptr) r.e[j] = R[at + j];
        }
      }
    }
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const uint4 w = rng((uint64_t)(i * (V / 4) + q));
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool keep = ws[j] >= thr && !none;
        // a dropped element contributes 0 whatever it holds (no inf * 0)
        const float v = keep ? elem_to_f32(x.e[4 * q + j]) : 0.0f;
        y.e[4 * q + j] = elem_from_f32<E>(R != nullptr ? fmaf(v, a.scale, elem_to_f32(r.e[4 * q + j])) : v * a.scale);
      }
    }
    if (ALIGNED && whole) {
      store_pack<E, V>(Y + at, y);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < a.n) Y[at + j] = y.e[j];
    }
  }
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
  spk::DropoutArgs a{};
  a.x = X;
  a.r = R;
  a.y = Y;
  a.n = n;
  a.seed = seed;
  a.offset = offset;
  a.key = key;
  a.threshold = (uint64_t)(p * 4294967296.0 + 0.5);
  a.scale = a.threshold <= 0xffffffffull ? (float)(1.0 / (1.0 - p)) : 0.0f;  // nothing kept: 0, not 0 * inf
  const bool aligned = spk::aligned_to(X, 16) && spk::aligned_to(R, 16) && spk::aligned_to(Y, 16);
  const int64_t vecs = spk::ceil_div(n, (int64_t)(16 / eb));
  const int64_t blocks = spk::min64(spk::ceil_div(vecs, 256), (int64_t)spk::sm_count() * 8);
  cudaStream_t st = (cudaStream_t)stream;
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    if (aligned)
      spk::dropout_kernel<E, true><<<(unsigned)blocks, 256, 0, st>>>(a);
    else
      spk::dropout_kernel<E, false><<<(unsigned)blocks, 256, 0, st>>>(a);
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
  return SPK_OK;
}
