// Group norm with an activation on channels-last tensors, and its backward
// pass.  X is [S, P, C] (S samples of P positions), the C channels form G
// groups of cg = C / G neighbours; per sample and group, over its n = P cg
// elements:
//   mean, var (biased),  xhat = (x - mean) / sqrt(var + eps),
//   z = xhat * weight[c] + bias[c],  y = act(z).
// Backward, with dz = gy act'(z) and dn = dz weight[c]:
//   dbias[c] = sum dz,  dweight[c] = sum dz xhat   (over samples and positions),
//   dx = rstd (dn - mean(dn) - xhat mean(dn xhat))  (means over the group).
// act' of the Heaviside activation is the sigmoid surrogate of spike_fn
// (slope 10).  The variance is never a difference of two large sums: parts
// carry (count, mean, sum of squares about their own mean) and are merged.
//
// Bound: HBM; x (and gy) read and y (dx) written.
#include "elem.cuh"

namespace spk {

struct GnArgs {
  const void* x;
  const void* gy;
  const float* weight;  // [C] or null (1)
  const float* bias;    // [C] or null (0)
  void* y;              // y, or dx in the backward pass
  float* mean;          // [S, G]
  float* rstd;          // [S, G]
  float* part;          // partial sums: [S, tiles, C, 2]
  float* coef;          // backward: [S, G, 2] mean(dn), mean(dn xhat)
  float* dweight;
  float* dbias;
  int64_t S, P;
  int C, G, cg;
  int rows, tiles;      // positions per tile, tiles per sample
  float eps, thr;
};

template <int ACT>
__device__ __forceinline__ float gn_act(float z, float thr) {
  if (ACT == SPK_ACT_HEAVISIDE) return z - thr > 0.0f ? 1.0f : 0.0f;
  if (ACT == SPK_ACT_SILU) return z * __fdividef(1.0f, 1.0f + expf(-z));
  return z;
}

// act'(z) gy
template <int ACT>
__device__ __forceinline__ float gn_act_grad(float z, float thr, float gy) {
  if (ACT == SPK_ACT_HEAVISIDE) {
    const float s = __fdividef(1.0f, 1.0f + expf(-10.0f * (z - thr)));
    return gy * s * (1.0f - s) * 10.0f;
  }
  if (ACT == SPK_ACT_SILU) {
    const float s = __fdividef(1.0f, 1.0f + expf(-z));
    return gy * (s * fmaf(z, 1.0f - s, 1.0f));
  }
  return gy;
}

struct Moments {
  float n, mean, m2;
};

__device__ __forceinline__ Moments merge(const Moments& a, const Moments& b) {
  Moments r;
  r.n = a.n + b.n;
  const float w = r.n > 0.0f ? __fdividef(b.n, r.n) : 0.0f;
  const float d = b.mean - a.mean;
  r.mean = fmaf(d, w, a.mean);
  r.m2 = a.m2 + b.m2 + d * d * a.n * w;
  return r;
}

constexpr int kGnThreads = 256;

// Partial moments of one channel over the rows of one tile: thread = channel
// (blockIdx.y tiles the channels), rows split over threadIdx.y.
template <typename E>
__global__ void __launch_bounds__(kGnThreads) gn_stats_kernel(GnArgs a) {
  __shared__ Moments sm[8][32];
  const int c = blockIdx.y * 32 + threadIdx.x;
  const int64_t tile = blockIdx.x, s = tile / a.tiles;
  const int64_t p0 = (tile - s * a.tiles) * a.rows, p1 = min64(p0 + a.rows, a.P);
  Moments m{0.0f, 0.0f, 0.0f};
  if (c < a.C) {
    const E* x = static_cast<const E*>(a.x) + (s * a.P) * a.C + c;
    for (int64_t p = p0 + threadIdx.y; p < p1; p += 8) {
      m.n += 1.0f;
      const float v = elem_to_f32(x[p * a.C]), d = v - m.mean;
      m.mean += __fdividef(d, m.n);
      m.m2 = fmaf(d, v - m.mean, m.m2);
    }
  }
  sm[threadIdx.y][threadIdx.x] = m;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.C) {
    for (int i = 1; i < 8; ++i) m = merge(m, sm[i][threadIdx.x]);
    float* out = a.part + (tile * a.C + c) * 2;
    out[0] = m.mean;
    out[1] = m.m2;
  }
}

__device__ __forceinline__ float gn_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp per (sample, group): merges the tiles' moments.
__global__ void __launch_bounds__(kGnThreads) gn_stats_finish_kernel(GnArgs a) {
  const int64_t u = (int64_t)blockIdx.x * (kGnThreads / 32) + (threadIdx.x >> 5);
  if (u >= a.S * a.G) return;
  const int lane = threadIdx.x & 31;
  const int64_t s = u / a.G, g = u - s * a.G, k = (int64_t)a.tiles * a.cg;
  const float total = (float)a.P * (float)a.cg;
  float sum = 0.0f, m2 = 0.0f;
  for (int64_t i = lane; i < k; i += 32) {
    const int64_t t = i / a.cg, c = g * a.cg + (i - t * a.cg);
    const float n = (float)(min64((t + 1) * a.rows, a.P) - t * a.rows);
    sum = fmaf(n, a.part[((s * a.tiles + t) * a.C + c) * 2], sum);
  }
  const float mean = gn_warp_sum(sum) / total;
  for (int64_t i = lane; i < k; i += 32) {
    const int64_t t = i / a.cg, c = g * a.cg + (i - t * a.cg);
    const float n = (float)(min64((t + 1) * a.rows, a.P) - t * a.rows);
    const float* part = a.part + ((s * a.tiles + t) * a.C + c) * 2;
    const float d = part[0] - mean;
    m2 += fmaf(n * d, d, part[1]);
  }
  const float var = gn_warp_sum(m2) / total;
  if (lane == 0) {
    a.mean[u] = mean;
    a.rstd[u] = rsqrtf(var + a.eps);
  }
}

template <typename E, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_apply_kernel(GnArgs a) {
  const int64_t n = a.S * a.P * a.C, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t row = i / a.C;
    const int c = (int)(i - row * a.C);
    const int64_t u = (row / a.P) * a.G + c / a.cg;
    const float w = a.weight != nullptr ? a.weight[c] : 1.0f, b = a.bias != nullptr ? a.bias[c] : 0.0f;
    const float xhat = (elem_to_f32(static_cast<const E*>(a.x)[i]) - a.mean[u]) * a.rstd[u];
    static_cast<E*>(a.y)[i] = elem_from_f32<E>(gn_act<ACT>(fmaf(xhat, w, b), a.thr));
  }
}

// Backward, per tile and channel: sum dz and sum dz xhat.
template <typename E, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_grad_sums_kernel(GnArgs a) {
  __shared__ float2 sm[8][32];
  const int c = blockIdx.y * 32 + threadIdx.x;
  const int64_t tile = blockIdx.x, s = tile / a.tiles;
  const int64_t p0 = (tile - s * a.tiles) * a.rows, p1 = min64(p0 + a.rows, a.P);
  float2 acc = make_float2(0.0f, 0.0f);
  if (c < a.C) {
    const float w = a.weight != nullptr ? a.weight[c] : 1.0f, b = a.bias != nullptr ? a.bias[c] : 0.0f;
    const float mean = a.mean[s * a.G + c / a.cg], rstd = a.rstd[s * a.G + c / a.cg];
    for (int64_t p = p0 + threadIdx.y; p < p1; p += 8) {
      const int64_t i = (s * a.P + p) * a.C + c;
      const float xhat = (elem_to_f32(static_cast<const E*>(a.x)[i]) - mean) * rstd;
      const float dz = gn_act_grad<ACT>(fmaf(xhat, w, b), a.thr, elem_to_f32(static_cast<const E*>(a.gy)[i]));
      acc.x += dz;
      acc.y = fmaf(dz, xhat, acc.y);
    }
  }
  sm[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  if (threadIdx.y == 0 && c < a.C) {
    for (int i = 1; i < 8; ++i) {
      acc.x += sm[i][threadIdx.x].x;
      acc.y += sm[i][threadIdx.x].y;
    }
    *reinterpret_cast<float2*>(a.part + (tile * a.C + c) * 2) = acc;
  }
}

// One warp per (sample, group): mean(dn) and mean(dn xhat).
__global__ void __launch_bounds__(kGnThreads) gn_grad_finish_kernel(GnArgs a) {
  const int64_t u = (int64_t)blockIdx.x * (kGnThreads / 32) + (threadIdx.x >> 5);
  if (u >= a.S * a.G) return;
  const int lane = threadIdx.x & 31;
  const int64_t s = u / a.G, g = u - s * a.G, k = (int64_t)a.tiles * a.cg;
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t i = lane; i < k; i += 32) {
    const int64_t t = i / a.cg, c = g * a.cg + (i - t * a.cg);
    const float w = a.weight != nullptr ? a.weight[c] : 1.0f;
    const float* part = a.part + ((s * a.tiles + t) * a.C + c) * 2;
    s1 = fmaf(w, part[0], s1);
    s2 = fmaf(w, part[1], s2);
  }
  s1 = gn_warp_sum(s1);
  s2 = gn_warp_sum(s2);
  if (lane == 0) {
    const float inv = 1.0f / ((float)a.P * (float)a.cg);
    a.coef[2 * u] = s1 * inv;
    a.coef[2 * u + 1] = s2 * inv;
  }
}

template <typename E, int ACT>
__global__ void __launch_bounds__(kGnThreads) gn_grad_apply_kernel(GnArgs a) {
  const int64_t n = a.S * a.P * a.C, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
    const int64_t row = i / a.C;
    const int c = (int)(i - row * a.C);
    const int64_t u = (row / a.P) * a.G + c / a.cg;
    const float w = a.weight != nullptr ? a.weight[c] : 1.0f, b = a.bias != nullptr ? a.bias[c] : 0.0f;
    const float rstd = a.rstd[u];
    const float xhat = (elem_to_f32(static_cast<const E*>(a.x)[i]) - a.mean[u]) * rstd;
    const float dz = gn_act_grad<ACT>(fmaf(xhat, w, b), a.thr, elem_to_f32(static_cast<const E*>(a.gy)[i]));
    static_cast<E*>(a.y)[i] = elem_from_f32<E>(rstd * (dz * w - a.coef[2 * u] - xhat * a.coef[2 * u + 1]));
  }
}

// dweight and dbias: the partial sums over all samples and tiles, in a fixed
// order (the same bits on every run).  32 channels per block, 32 threads each.
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(GnArgs a) {
  __shared__ float2 sm[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float2 acc = make_float2(0.0f, 0.0f);
  if (c < a.C) {
    const int64_t rows = a.S * a.tiles;
    for (int64_t r = threadIdx.y; r < rows; r += 32) {
      const float2 v = *reinterpret_cast<const float2*>(a.part + (r * a.C + c) * 2);
      acc.x += v.x;
      acc.y += v.y;
    }
  }
  sm[threadIdx.y][threadIdx.x] = acc;
  __syncthreads();
  const float2 v = sm[threadIdx.x][threadIdx.y];  // warp y: the 32 parts of channel y
  const float db = gn_warp_sum(v.x), dw = gn_warp_sum(v.y);
  const int co = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && co < a.C) {
    if (a.dbias != nullptr) a.dbias[co] = db;
    if (a.dweight != nullptr) a.dweight[co] = dw;
  }
}

// Positions per tile: enough tiles to fill the GPU, at least 64 positions each
// so that the partial sums stay small beside the tensor.
static void gn_tiling(int64_t S, int64_t P, int C, int* rows, int* tiles) {
  const int64_t want = ceil_div(148 * 8, max64(S * ceil_div(C, 32), 1));
  const int64_t r = max64(64, max64(ceil_div(P, max64(want, 1)), ceil_div(P, 65535)));
  *rows = (int)min64(r, max64(P, 1));
  *tiles = (int)ceil_div(max64(P, 1), *rows);
}

static size_t gn_part_bytes(int64_t S, int64_t P, int C) {
  int rows, tiles;
  gn_tiling(S, P, C, &rows, &tiles);
  return align_up((size_t)S * tiles * C * 2 * sizeof(float), 256);
}

static int gn_check(int dtype, int64_t S, int64_t P, int C, int G, int act, size_t* eb) {
  SPK_REQUIRE(S >= 0 && P >= 0 && C >= 1 && G >= 1, "invalid shape (S=%lld, P=%lld, C=%d, G=%d)", (long long)S,
              (long long)P, C, G);
  SPK_REQUIRE(C % G == 0, "C=%d is not a multiple of the %d groups", C, G);
  *eb = elem_bytes(dtype);
  SPK_REQUIRE(*eb != 0, "unknown element type %d", dtype);
  SPK_REQUIRE(act == SPK_ACT_NONE || act == SPK_ACT_HEAVISIDE || act == SPK_ACT_SILU,
              "unknown group norm activation %d", act);
  SPK_REQUIRE(C <= (1 << 20) && P < (1ll << 31) && S < (1ll << 31) && (P == 0 || S < (1ll << 42) / ((int64_t)C * P)),
              "shape too large (S=%lld, P=%lld, C=%d)", (long long)S, (long long)P, C);
  int rows, tiles;
  gn_tiling(S, P, C, &rows, &tiles);
  SPK_REQUIRE(S * tiles < (1ll << 31), "too many positions (S=%lld, P=%lld)", (long long)S, (long long)P);
  return SPK_OK;
}

template <typename F>
inline void with_gn_act(int act, F&& f) {
  if (act == SPK_ACT_HEAVISIDE)
    f(std::integral_constant<int, SPK_ACT_HEAVISIDE>{});
  else if (act == SPK_ACT_SILU)
    f(std::integral_constant<int, SPK_ACT_SILU>{});
  else
    f(std::integral_constant<int, SPK_ACT_NONE>{});
}

}  // namespace spk

extern "C" size_t spk_group_norm_workspace_bytes(int64_t S, int64_t P, int C, int G) {
  if (S <= 0 || P <= 0 || C <= 0 || G <= 0) return 0;
  return spk::gn_part_bytes(S, P, C) + (size_t)S * G * 2 * sizeof(float);
}

extern "C" int spk_group_norm_act(const void* X, int dtype, int64_t S, int64_t P, int C, int G, const float* weight,
                                  const float* bias, float eps, int act, float thr, void* Y, float* mean, float* rstd,
                                  void* workspace, size_t workspace_bytes, spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::gn_check(dtype, S, P, C, G, act, &eb)) return rc;
  SPK_REQUIRE(eps >= 0.0f, "eps must be non-negative");
  if (S == 0 || P == 0) return SPK_OK;
  SPK_REQUIRE(X != nullptr && Y != nullptr, "X and Y must be non-null");
  SPK_REQUIRE((mean == nullptr) == (rstd == nullptr), "mean and rstd go together");
  SPK_REQUIRE(spk::aligned_to(X, eb) && spk::aligned_to(Y, eb) && spk::aligned_to(weight, 4) &&
                  spk::aligned_to(bias, 4) && spk::aligned_to(mean, 4) && spk::aligned_to(rstd, 4),
              "tensors must be aligned to their elements");
  if (workspace == nullptr || workspace_bytes < spk_group_norm_workspace_bytes(S, P, C, G))
    return spk::fail(SPK_EWORKSPACE, "group norm needs a workspace of %zu bytes",
                     spk_group_norm_workspace_bytes(S, P, C, G));
  SPK_REQUIRE(spk::aligned_to(workspace, 16), "the workspace must be 16-byte aligned");
  spk::GnArgs a{};
  a.x = X;
  a.weight = weight;
  a.bias = bias;
  a.y = Y;
  a.part = static_cast<float*>(workspace);
  float* tail = reinterpret_cast<float*>(static_cast<char*>(workspace) + spk::gn_part_bytes(S, P, C));
  a.mean = mean != nullptr ? mean : tail;
  a.rstd = rstd != nullptr ? rstd : tail + S * G;
  a.S = S;
  a.P = P;
  a.C = C;
  a.G = G;
  a.cg = C / G;
  a.eps = eps;
  a.thr = thr;
  spk::gn_tiling(S, P, C, &a.rows, &a.tiles);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 tgrid((unsigned)(S * a.tiles), (unsigned)spk::ceil_div(C, 32)), tblock(32, 8);
  const unsigned ugrid = (unsigned)spk::ceil_div(S * G, spk::kGnThreads / 32);
  const unsigned egrid = (unsigned)spk::min64(spk::ceil_div(S * P * C, spk::kGnThreads), spk::sm_count() * 16);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    spk::gn_stats_kernel<E><<<tgrid, tblock, 0, st>>>(a);
    spk::gn_stats_finish_kernel<<<ugrid, spk::kGnThreads, 0, st>>>(a);
    spk::with_gn_act(act, [&](auto ac) {
      spk::gn_apply_kernel<E, decltype(ac)::value><<<egrid, spk::kGnThreads, 0, st>>>(a);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(3);
  return SPK_OK;
}

extern "C" int spk_group_norm_act_backward(const void* X, const void* GY, int dtype, int64_t S, int64_t P, int C,
                                           int G, const float* weight, const float* bias, const float* mean,
                                           const float* rstd, int act, float thr, void* DX, float* dweight,
                                           float* dbias, void* workspace, size_t workspace_bytes,
                                           spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::gn_check(dtype, S, P, C, G, act, &eb)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  SPK_REQUIRE(spk::aligned_to(dweight, 4) && spk::aligned_to(dbias, 4), "tensors must be aligned to their elements");
  if (S == 0 || P == 0) {  // no positions: sums over nothing
    if (dweight != nullptr) SPK_CUDA_TRY(cudaMemsetAsync(dweight, 0, (size_t)C * sizeof(float), st));
    if (dbias != nullptr) SPK_CUDA_TRY(cudaMemsetAsync(dbias, 0, (size_t)C * sizeof(float), st));
    return SPK_OK;
  }
  SPK_REQUIRE(X != nullptr && GY != nullptr && mean != nullptr && rstd != nullptr && DX != nullptr,
              "X, GY, mean, rstd and DX must be non-null");
  SPK_REQUIRE(spk::aligned_to(X, eb) && spk::aligned_to(GY, eb) && spk::aligned_to(DX, eb) &&
                  spk::aligned_to(weight, 4) && spk::aligned_to(bias, 4) && spk::aligned_to(mean, 4) &&
                  spk::aligned_to(rstd, 4),
              "tensors must be aligned to their elements");
  if (workspace == nullptr || workspace_bytes < spk_group_norm_workspace_bytes(S, P, C, G))
    return spk::fail(SPK_EWORKSPACE, "group norm needs a workspace of %zu bytes",
                     spk_group_norm_workspace_bytes(S, P, C, G));
  SPK_REQUIRE(spk::aligned_to(workspace, 16), "the workspace must be 16-byte aligned");
  spk::GnArgs a{};
  a.x = X;
  a.gy = GY;
  a.weight = weight;
  a.bias = bias;
  a.y = DX;
  a.mean = const_cast<float*>(mean);
  a.rstd = const_cast<float*>(rstd);
  a.part = static_cast<float*>(workspace);
  a.coef = reinterpret_cast<float*>(static_cast<char*>(workspace) + spk::gn_part_bytes(S, P, C));
  a.dweight = dweight;
  a.dbias = dbias;
  a.S = S;
  a.P = P;
  a.C = C;
  a.G = G;
  a.cg = C / G;
  a.thr = thr;
  spk::gn_tiling(S, P, C, &a.rows, &a.tiles);
  const dim3 tgrid((unsigned)(S * a.tiles), (unsigned)spk::ceil_div(C, 32)), tblock(32, 8);
  const unsigned ugrid = (unsigned)spk::ceil_div(S * G, spk::kGnThreads / 32);
  const unsigned egrid = (unsigned)spk::min64(spk::ceil_div(S * P * C, spk::kGnThreads), spk::sm_count() * 16);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    spk::with_gn_act(act, [&](auto ac) {
      constexpr int ACT = decltype(ac)::value;
      spk::gn_grad_sums_kernel<E, ACT><<<tgrid, tblock, 0, st>>>(a);
      spk::gn_grad_finish_kernel<<<ugrid, spk::kGnThreads, 0, st>>>(a);
      spk::gn_grad_apply_kernel<E, ACT><<<egrid, spk::kGnThreads, 0, st>>>(a);
      spk::gn_param_grad_kernel<<<(unsigned)spk::ceil_div(C, 32), dim3(32, 32), 0, st>>>(a);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(4);
  return SPK_OK;
}
