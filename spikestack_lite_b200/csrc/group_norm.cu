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
// Bound: HBM, x (and gy) read and y (dx) written, for fp32; the issue of
// instructions (two for the MUFU unit among some 20 per element and pass with
// SiLU) for 16-bit tensors.  Two forms.  Resident: a block or a cluster keeps
// what it normalises in shared memory and every tensor crosses HBM once.
// Tiled: samples beyond that pass twice, sums first.  Measured, SiLU:
//   resident  256x1024x512 fp32 forward 170 us (97 % of what its bytes need at the
//             measured HBM rate), backward 361 us (68 %); bf16 117 / 269 us
//   tiled     4x32768x512 bf16 93 us forward, 149 us backward (66 and 69 % of the
//             bytes of both passes)
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
  int tpr, rpp, threads;  // threads side by side and rows at once in a block
  int held, split;      // bytes of the tensors that a block holds, blocks per sample and groups (resident)
  int k, rows, tiles;   // groups per block (resident); positions per block; blocks per sample (and position share)
  int64_t parts;        // rows of `part`
  float eps, thr;
};

constexpr int kGnThreads = 256;

// sigmoid with the hardware's exponential: with u = 2^-24, off by 4 u of the
// exponential itself and 1.5 |z| u of its argument's rounding, as much as the
// rounding of z lets it be off anyway.  256x1024x512 fp32 takes 170 us forward
// and 361 us backward with it, 178 and 388 with expf.
__device__ __forceinline__ float gn_sigmoid(float z) { return rcp_fast(1.0f + ex2_fast(z * -1.4426950409f)); }

template <int ACT>
__device__ __forceinline__ float gn_act(float z, float thr) {
  if (ACT == SPK_ACT_HEAVISIDE) return z - thr > 0.0f ? 1.0f : 0.0f;
  if (ACT == SPK_ACT_SILU) return z * gn_sigmoid(z);
  return z;
}

// act'(z) gy
template <int ACT>
__device__ __forceinline__ float gn_act_grad(float z, float thr, float gy) {
  if (ACT == SPK_ACT_HEAVISIDE) {
    const float s = gn_sigmoid(10.0f * (z - thr));
    return gy * s * (1.0f - s) * 10.0f;
  }
  if (ACT == SPK_ACT_SILU) {
    const float s = gn_sigmoid(z);
    return gy * (s * fmaf(z, 1.0f - s, 1.0f));
  }
  return gy;
}

__device__ __forceinline__ float gn_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A block's threads over a tile: V neighbouring channels each, `tpr` threads
// side by side, `rpp` rows at once (the rest of the block idles).
struct GnSpot {
  int cv, r;  // the thread's first channel within the tile's columns, its first row
  bool live;
};

__device__ __forceinline__ GnSpot gn_spot(int V, int tpr, int rpp) {
  GnSpot q;
  q.r = (int)threadIdx.x / tpr;
  q.cv = ((int)threadIdx.x - q.r * tpr) * V;
  q.live = q.r < rpp;
  return q;
}

// Constants of the thread's V channels, which lie in M groups at most (M = 1:
// in one): with d = x - mean, z = d (rstd weight) + bias.
template <int V, int M>
struct GnAffine {
  float mean[M], rstd[M], a[V], b[V];
};

// f(j, group) for the channels c .. c + V - 1 of groups of cg channels.
template <int V, int M, typename F>
__device__ __forceinline__ void gn_groups(int c, int cg, F&& f) {
  int g = c / cg, left = cg - (c - g * cg);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (M > 1 && left == 0) {
      ++g;
      left = cg;
    }
    f(j, g);
    --left;
  }
}

template <int V, int M>
__device__ __forceinline__ void gn_affine(const GnArgs& a, int c0, GnAffine<V, M>* f) {  // mean and rstd are set
#pragma unroll
  for (int j = 0; j < V; ++j) {
    f->a[j] = f->rstd[M > 1 ? j : 0] * (a.weight != nullptr ? a.weight[c0 + j] : 1.0f);
    f->b[j] = a.bias != nullptr ? a.bias[c0 + j] : 0.0f;
  }
}

template <int V, int M>
__device__ __forceinline__ void gn_affine(const GnArgs& a, int64_t s, int c0, GnAffine<V, M>* f) {
  gn_groups<V, M>(c0, a.cg, [&](int j, int g) {
    if (M > 1 || j == 0) {
      f->mean[M > 1 ? j : 0] = a.mean[s * a.G + g];
      f->rstd[M > 1 ? j : 0] = a.rstd[s * a.G + g];
    }
  });
  gn_affine<V, M>(a, c0, f);
}

template <typename E, int ACT, int V, int M>
__device__ __forceinline__ Pack<E, V> gn_forward(const Pack<E, V>& x, const GnAffine<V, M>& f, float thr) {
  float y[V];
#pragma unroll
  for (int j = 0; j < V; ++j)
    y[j] = gn_act<ACT>(fmaf(elem_to_f32(x.e[j]) - f.mean[M > 1 ? j : 0], f.a[j], f.b[j]), thr);
  return pack_f32<E, V>(y);
}

// dz and d of one element.
template <typename E, int ACT, int V, int M>
__device__ __forceinline__ float gn_dz(const Pack<E, V>& x, const Pack<E, V>& gy, const GnAffine<V, M>& f, int j,
                                       float thr, float* d) {
  *d = elem_to_f32(x.e[j]) - f.mean[M > 1 ? j : 0];
  return gn_act_grad<ACT>(fmaf(*d, f.a[j], f.b[j]), thr, elem_to_f32(gy.e[j]));
}

// What a group's means m = (mean(dn), mean(dn xhat)) do to dx:
// dx = rstd (dn - m.x - xhat m.y) = dz (rstd weight) + d k.y + k.x.
__device__ __forceinline__ float2 gn_pull(float2 m, float rstd) {
  return make_float2(-rstd * m.x, -rstd * rstd * m.y);
}

template <typename E, int ACT, int V, int M>
__device__ __forceinline__ Pack<E, V> gn_backward(const Pack<E, V>& x, const Pack<E, V>& gy,
                                                  const GnAffine<V, M>& f, const float2 (&k)[M], float thr) {
  float o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float d;
    const float dz = gn_dz<E, ACT, V, M>(x, gy, f, j, thr, &d);
    const float2 kj = k[M > 1 ? j : 0];
    o[j] = fmaf(dz, f.a[j], fmaf(d, kj.y, kj.x));
  }
  return pack_f32<E, V>(o);
}

// ---- resident form: a block, or a cluster of `split` blocks with a share of
// the positions each, holds a sample's k groups in shared memory, so x (and gy)
// cross HBM once.  Every thread copies the packs (16 bytes) that it will read
// itself; what waits is memory, not registers, so some 30 warps share an SM.
// The blocks of a cluster read each other's group sums, in the order of ranks.
struct GnShare {
  int64_t s, p0;  // sample, first position
  int P, rank;    // positions
  int g0, ng;     // groups

  __device__ __forceinline__ explicit GnShare(const GnArgs& a) {
    const unsigned unit = blockIdx.x / (unsigned)a.split, sample = unit / (unsigned)a.tiles;  // below 2^31
    rank = (int)(blockIdx.x - unit * a.split);
    s = sample;
    g0 = (int)(unit - sample * a.tiles) * a.k;
    ng = min(a.k, a.G - g0);
    p0 = (int64_t)rank * a.rows;
    P = positions(a, rank);
  }
  __device__ __forceinline__ static int positions(const GnArgs& a, int rank) {
    return max(min((int)a.P - rank * a.rows, a.rows), 0);  // split * rows < P + split
  }
};

template <typename E, int V>
struct GnPacks {
  E* slot;  // the thread's packs of one tensor, blockDim packs apart
  int rows;

  __device__ __forceinline__ GnPacks(unsigned char* smem, int rows_)
      : slot(reinterpret_cast<E*>(smem) + threadIdx.x * V), rows(rows_) {}
  __device__ __forceinline__ void ask(const E* p, int64_t step) const {
    E* to = slot;
    for (int i = 0; i < rows; ++i, p += step, to += blockDim.x * V)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(p) : "memory");
  }
  __device__ __forceinline__ Pack<E, V> get(int i) const { return load_pack<E, V>(slot + i * (int)(blockDim.x * V)); }
};
__device__ __forceinline__ void gn_wait_packs() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// WHOLE: every pack lies in one group (cg is a multiple of V); a part is then
// the moments of one thread, else those of one channel of one thread.
template <typename E, int ACT, bool WHOLE>
__global__ void __launch_bounds__(512, 2) gn_resident_kernel(GnArgs a) {
  constexpr int V = 16 / (int)sizeof(E), M = WHOLE ? 1 : V;
  extern __shared__ __align__(16) unsigned char gn_smem[];
  const GnShare h(a);
  const int width = h.ng * a.cg;
  GnSpot q = gn_spot(V, a.tpr, a.rpp);
  q.live = q.live && q.cv < width;
  const int least = h.P / a.rpp, extra = h.P - least * a.rpp;
  const int rows = q.live ? least + (q.r < extra ? 1 : 0) : 0, c0 = h.g0 * a.cg + q.cv;
  const int64_t at = (h.s * a.P + h.p0 + q.r) * a.C + c0, step = (int64_t)a.rpp * a.C;
  const GnPacks<E, V> x(gn_smem, rows);
  x.ask(static_cast<const E*>(a.x) + at, step);
  float2* const part = reinterpret_cast<float2*>(gn_smem + a.held);  // [groups][parts] mean, sum of squares about it
  const int per_row = WHOLE ? a.cg / V : a.cg, parts = a.rpp * per_row;  // of one group, row by row
  float2* const stat = part + a.k * parts;                              // [k]
  gn_wait_packs();
  if (q.live) {
    float sum[M], m2[M];
#pragma unroll
    for (int j = 0; j < M; ++j) sum[j] = m2[j] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < rows; ++i) {
      const Pack<E, V> p = x.get(i);
      float all = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (M > 1)
          sum[M > 1 ? j : 0] += elem_to_f32(p.e[j]);
        else
          all += elem_to_f32(p.e[j]);
      }
      if (M == 1) sum[0] += all;
    }
    const float inv = rows > 0 ? __fdividef(1.0f, (float)(rows * (WHOLE ? V : 1))) : 0.0f;
#pragma unroll
    for (int j = 0; j < M; ++j) sum[j] *= inv;
#pragma unroll 4
    for (int i = 0; i < rows; ++i) {
      const Pack<E, V> p = x.get(i);
      float all = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = elem_to_f32(p.e[j]) - sum[M > 1 ? j : 0];
        if (M > 1)
          m2[M > 1 ? j : 0] = fmaf(d, d, m2[M > 1 ? j : 0]);
        else
          all = fmaf(d, d, all);
      }
      if (M == 1) m2[0] += all;
    }
    gn_groups<V, M>(q.cv, a.cg, [&](int j, int g) {
      if (M > 1 || j == 0)
        part[g * parts + q.r * per_row + (q.cv + j - g * a.cg) / (WHOLE ? V : 1)] =
            make_float2(sum[M > 1 ? j : 0], m2[M > 1 ? j : 0]);
    });
  }
  __syncthreads();
  // one warp per group; the first `more` parts have a row more than the rest
  const int lane = threadIdx.x & 31, more = extra * per_row;
  const float mine = (float)h.P * (float)a.cg, total = (float)a.P * (float)a.cg;
  const float n_more = (float)((least + 1) * (WHOLE ? V : 1)), n_less = (float)(least * (WHOLE ? V : 1));
  for (int g = threadIdx.x >> 5; g < h.ng; g += blockDim.x / 32) {
    float sum = 0.0f, m2 = 0.0f;
    for (int i = lane; i < parts; i += 32) sum = fmaf(i < more ? n_more : n_less, part[g * parts + i].x, sum);
    const float mean = h.P > 0 ? gn_warp_sum(sum) / mine : 0.0f;
    for (int i = lane; i < parts; i += 32) {
      const float2 v = part[g * parts + i];
      const float d = v.x - mean;
      m2 += fmaf((i < more ? n_more : n_less) * d, d, v.y);
    }
    m2 = gn_warp_sum(m2);
    if (lane == 0) stat[g] = make_float2(mean, m2);
  }
  float2* const own = stat + a.k;  // [k] mean and rstd
  if (a.split > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int g = threadIdx.x; g < h.ng; g += blockDim.x) {
    float2 m = stat[g];
    if (a.split > 1) {
      float sum = 0.0f, m2 = 0.0f;
      for (int r = 0; r < a.split; ++r)
        sum = fmaf((float)GnShare::positions(a, r) * (float)a.cg, cluster_load(stat + g, r).x, sum);
      const float mean = sum / total;
      for (int r = 0; r < a.split; ++r) {
        const float2 v = cluster_load(stat + g, r);
        const float d = v.x - mean;
        m2 += fmaf((float)GnShare::positions(a, r) * (float)a.cg * d, d, v.y);
      }
      m = make_float2(mean, m2);
    }
    m.y = rsqrtf(m.y / total + a.eps);
    own[g] = m;
    if (a.mean != nullptr && h.rank == 0) {
      a.mean[h.s * a.G + h.g0 + g] = m.x;
      a.rstd[h.s * a.G + h.g0 + g] = m.y;
    }
  }
  if (a.split > 1) cluster_arrive();
  __syncthreads();
  if (q.live) {
    GnAffine<V, M> f;
    gn_groups<V, M>(q.cv, a.cg, [&](int j, int g) {
      if (M > 1 || j == 0) {
        f.mean[M > 1 ? j : 0] = own[g].x;
        f.rstd[M > 1 ? j : 0] = own[g].y;
      }
    });
    gn_affine<V, M>(a, c0, &f);
    E* y = static_cast<E*>(a.y) + at;
#pragma unroll 2
    for (int i = 0; i < rows; ++i, y += step) store_pack<E, V>(y, gn_forward<E, ACT, V, M>(x.get(i), f, a.thr));
  }
  if (a.split > 1) cluster_wait();  // stat is read by the others
}

// Sums over the rows of part [rpp][width], by the whole block and in a fixed
// order: `some` [segments][width] (at most one entry per thread), then sums [width].
__device__ __forceinline__ void gn_channel_sums(const float2* part, int rpp, int width, float2* some, float2* sums) {
  const int threads = blockDim.x, segments = max(1, min(rpp, threads / width));
  for (int i = threadIdx.x; i < segments * width; i += threads) {
    const int seg = i / width, c = i - seg * width;
    float2 v = make_float2(0.0f, 0.0f);
    for (int r = seg; r < rpp; r += segments) {
      v.x += part[r * width + c].x;
      v.y += part[r * width + c].y;
    }
    (segments > 1 ? some : sums)[i] = v;
  }
  __syncthreads();
  if (segments > 1) {
    for (int c = threadIdx.x; c < width; c += threads) {
      float2 v = some[c];
      for (int i = 1; i < segments; ++i) {
        v.x += some[i * width + c].x;
        v.y += some[i * width + c].y;
      }
      sums[c] = v;
    }
    __syncthreads();
  }
}

template <typename E, int ACT, bool WHOLE>
__global__ void __launch_bounds__(512, 2) gn_resident_backward_kernel(GnArgs a) {
  constexpr int V = 16 / (int)sizeof(E), M = WHOLE ? 1 : V;
  extern __shared__ __align__(16) unsigned char gn_smem[];
  grid_dependents_may_start();
  const GnShare h(a);
  const int width = h.ng * a.cg;
  GnSpot q = gn_spot(V, a.tpr, a.rpp);
  q.live = q.live && q.cv < width;
  const int rows = q.live ? (max(h.P - q.r, 0) + a.rpp - 1) / a.rpp : 0, c0 = h.g0 * a.cg + q.cv;
  const int64_t at = (h.s * a.P + h.p0 + q.r) * a.C + c0, step = (int64_t)a.rpp * a.C;
  const GnPacks<E, V> x(gn_smem, rows), gy(gn_smem + a.held / 2, rows);
  x.ask(static_cast<const E*>(a.x) + at, step);
  gy.ask(static_cast<const E*>(a.gy) + at, step);
  // where a warp holds whole rows, its lanes first add up theirs
  const bool fold = 32 % a.tpr == 0;
  const int sets = fold ? (int)blockDim.x / 32 : a.rpp;
  float2* const part = reinterpret_cast<float2*>(gn_smem + a.held);  // [sets][width] sums of dz and dz xhat
  float2* const sums = part + sets * a.k * a.cg;                     // [width]
  float2* const coef = sums + a.k * a.cg;                            // [k]
  GnAffine<V, M> f;
  if (q.live) gn_affine<V, M>(a, h.s, c0, &f);
  gn_wait_packs();
  float s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.0f;
  if (q.live) {
#pragma unroll 2
    for (int i = 0; i < rows; ++i) {
      const Pack<E, V> xv = x.get(i), gv = gy.get(i);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float d;
        const float dz = gn_dz<E, ACT, V, M>(xv, gv, f, j, a.thr, &d);
        s1[j] += dz;
        s2[j] = fmaf(dz, d, s2[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s2[j] *= f.rstd[M > 1 ? j : 0];
  }
  if (fold) {
    for (int o = a.tpr; o < 32; o *= 2) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s1[j] += __shfl_xor_sync(0xffffffffu, s1[j], o);
        s2[j] += __shfl_xor_sync(0xffffffffu, s2[j], o);
      }
    }
  }
  if (q.live && (!fold || (int)(threadIdx.x & 31) < a.tpr)) {
    float2* const to = part + (fold ? (int)threadIdx.x / 32 : q.r) * width + q.cv;
#pragma unroll
    for (int j = 0; j < V; ++j) to[j] = make_float2(s1[j], s2[j]);
  }
  __syncthreads();
  float2* const own = coef + a.k;  // [k] this block's sums of dn and dn xhat
  gn_channel_sums(part, sets, width, own + a.k, sums);
  const int lane = threadIdx.x & 31;
  const float inv = 1.0f / ((float)a.P * (float)a.cg);
  for (int g = threadIdx.x >> 5; g < h.ng; g += blockDim.x / 32) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int i = lane; i < a.cg; i += 32) {
      const float w = a.weight != nullptr ? a.weight[(h.g0 + g) * a.cg + i] : 1.0f;
      s1 = fmaf(w, sums[g * a.cg + i].x, s1);
      s2 = fmaf(w, sums[g * a.cg + i].y, s2);
    }
    s1 = gn_warp_sum(s1);
    s2 = gn_warp_sum(s2);
    if (lane == 0) own[g] = make_float2(s1, s2);
  }
  if (a.part != nullptr)
    for (int c = threadIdx.x; c < width; c += blockDim.x)
      *reinterpret_cast<float2*>(a.part + ((h.s * a.split + h.rank) * a.C + h.g0 * a.cg + c) * 2) = sums[c];
  if (a.split > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int g = threadIdx.x; g < h.ng; g += blockDim.x) {
    float2 m = own[g];
    if (a.split > 1) {
      m = make_float2(0.0f, 0.0f);
      for (int r = 0; r < a.split; ++r) {
        const float2 v = cluster_load(own + g, r);
        m.x += v.x;
        m.y += v.y;
      }
    }
    coef[g] = make_float2(m.x * inv, m.y * inv);
  }
  if (a.split > 1) cluster_arrive();
  __syncthreads();
  if (q.live) {
    E* dx = static_cast<E*>(a.y) + at;
    float2 k[M];
    gn_groups<V, M>(q.cv, a.cg, [&](int j, int g) {
      if (M > 1 || j == 0) k[M > 1 ? j : 0] = gn_pull(coef[g], f.rstd[M > 1 ? j : 0]);
    });
#pragma unroll 2
    for (int i = 0; i < rows; ++i, dx += step)
      store_pack<E, V>(dx, gn_backward<E, ACT, V, M>(x.get(i), gy.get(i), f, k, a.thr));
  }
  if (a.split > 1) cluster_wait();  // own is read by the others
}

// ---- tiled form: samples larger than a block holds.  Tiles of `rows`
// positions; a tile's moments (sums) per channel, the join per sample and
// group, then the apply pass, whose tiles run from the last to the first, so
// that it finds in L2 what the first pass read last.
struct GnTile {
  int64_t s, p0;
  int rows, c0;  // positions, the thread's first channel
  bool live;
};

template <int V>
__device__ __forceinline__ GnTile gn_tile(const GnArgs& a, int64_t tile, const GnSpot& q) {
  GnTile t;
  const unsigned at = (unsigned)tile, sample = at / (unsigned)a.tiles;  // below 2^31
  t.s = sample;
  t.p0 = (int64_t)(at - sample * a.tiles) * a.rows;
  t.rows = (int)min64(a.rows, a.P - t.p0);
  t.c0 = (int)blockIdx.y * a.tpr * V + q.cv;
  t.live = q.live && t.c0 < a.C;
  return t;
}

constexpr int kGnBatch = 4, kGnGradBatch = 2;  // rows in flight per thread (of one tensor, of two)

template <typename E, int V>
__global__ void __launch_bounds__(kGnThreads, 4) gn_stats_kernel(GnArgs a) {
  extern __shared__ __align__(16) unsigned char gn_smem[];
  float2* const part = reinterpret_cast<float2*>(gn_smem);  // [rpp][tpr V]
  const GnSpot q = gn_spot(V, a.tpr, a.rpp);
  const GnTile t = gn_tile<V>(a, blockIdx.x, q);
  grid_dependents_may_start();
  float mean[V], m2[V], n = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) mean[j] = m2[j] = 0.0f;
  if (t.live) {
    const E* x = static_cast<const E*>(a.x) + (t.s * a.P + t.p0) * a.C + t.c0;
    for (int p = q.r; p < t.rows; p += kGnBatch * a.rpp) {
      Pack<E, V> v[kGnBatch];
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < kGnBatch; ++i)
        if (p + i * a.rpp < t.rows) {
          v[i] = load_pack<E, V>(x + (int64_t)(p + i * a.rpp) * a.C);
          m += 1.0f;
        }
      const float inv = __fdividef(1.0f, m), w = __fdividef(m, n + m), nw = n * w;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kGnBatch; ++i)
          if (p + i * a.rpp < t.rows) sum += elem_to_f32(v[i].e[j]);
        const float mb = sum * inv, d = mb - mean[j];
        m2[j] = fmaf(d * d, nw, m2[j]);
#pragma unroll
        for (int i = 0; i < kGnBatch; ++i)
          if (p + i * a.rpp < t.rows) {
            const float e = elem_to_f32(v[i].e[j]) - mb;
            m2[j] = fmaf(e, e, m2[j]);
          }
        mean[j] = fmaf(d, w, mean[j]);
      }
      n += m;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) part[q.r * a.tpr * V + q.cv + j] = make_float2(mean[j], m2[j]);
  }
  __syncthreads();
  // the row threads' parts of one channel, in a fixed order
  const int width = min(a.tpr * V, a.C - (int)blockIdx.y * a.tpr * V);
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float2 v = part[c];
    float cnt = (float)((t.rows + a.rpp - 1) / a.rpp);
    for (int r = 1; r < a.rpp && r < t.rows; ++r) {
      const float2 o = part[r * a.tpr * V + c];
      const float k = (float)((t.rows - r + a.rpp - 1) / a.rpp), w = __fdividef(k, cnt + k), d = o.x - v.x;
      v.x = fmaf(d, w, v.x);
      v.y += fmaf(d * d, cnt * w, o.y);
      cnt += k;
    }
    *reinterpret_cast<float2*>(a.part + ((int64_t)blockIdx.x * a.C + blockIdx.y * a.tpr * V + c) * 2) = v;
  }
}

template <int THREADS>
__device__ __forceinline__ float gn_block_sum(float v, float* sm) {
  v = gn_warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = 0.0f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) r += sm[i];
  __syncthreads();
  return r;
}

// The parts of one group, every kGnThreads-th from this thread's on: f(tile, channel).
template <typename F>
__device__ __forceinline__ void gn_each_part(const GnArgs& a, F&& f) {
  const int down = kGnThreads / a.cg, right = kGnThreads - down * a.cg;
  int t = (int)threadIdx.x / a.cg, c = (int)threadIdx.x - t * a.cg;
#pragma unroll 4
  for (; t < a.tiles; t += down) {
    f(t, c);
    c += right;
    if (c >= a.cg) {
      c -= a.cg;
      ++t;
    }
  }
}

// One block per (sample, group): joins the tiles' moments.
__global__ void __launch_bounds__(kGnThreads) gn_stats_finish_kernel(GnArgs a) {
  __shared__ float sm[kGnThreads / 32];
  grid_dependents_may_start();
  grid_wait_for_previous();
  const unsigned u = blockIdx.x, sample = u / (unsigned)a.G;
  const int64_t s = sample, g = u - sample * a.G;
  const float2* part = reinterpret_cast<const float2*>(a.part) + s * a.tiles * a.C + g * a.cg;
  const float total = (float)a.P * (float)a.cg, rows = (float)a.rows;
  const float tail = (float)(int)(a.P - (int64_t)(a.tiles - 1) * a.rows);  // rows of the last tile
  float sum = 0.0f, m2 = 0.0f;
  gn_each_part(a, [&](int t, int c) {
    sum = fmaf(t + 1 < a.tiles ? rows : tail, part[(int64_t)t * a.C + c].x, sum);
  });
  const float mean = gn_block_sum<kGnThreads>(sum, sm) / total;
  gn_each_part(a, [&](int t, int c) {
    const float2 v = part[(int64_t)t * a.C + c];
    const float d = v.x - mean;
    m2 += fmaf((t + 1 < a.tiles ? rows : tail) * d, d, v.y);
  });
  const float var = gn_block_sum<kGnThreads>(m2, sm) / total;
  if (threadIdx.x == 0) {
    a.mean[u] = mean;
    a.rstd[u] = rsqrtf(var + a.eps);
  }
}

template <typename E, int ACT, int V, int M>
__global__ void __launch_bounds__(kGnThreads, 4) gn_apply_kernel(GnArgs a) {
  const GnSpot q = gn_spot(V, a.tpr, a.rpp);
  const GnTile t = gn_tile<V>(a, gridDim.x - 1 - (int64_t)blockIdx.x, q);
  grid_dependents_may_start();
  grid_wait_for_previous();
  if (!t.live) return;
  GnAffine<V, M> f;
  gn_affine<V, M>(a, t.s, t.c0, &f);
  const int64_t at = (t.s * a.P + t.p0) * a.C + t.c0;
  const E* x = static_cast<const E*>(a.x) + at;
  E* y = static_cast<E*>(a.y) + at;
  for (int p = q.r; p < t.rows; p += kGnBatch * a.rpp) {
    Pack<E, V> v[kGnBatch];
#pragma unroll
    for (int i = 0; i < kGnBatch; ++i)
      if (p + i * a.rpp < t.rows) v[i] = load_pack<E, V>(x + (int64_t)(p + i * a.rpp) * a.C);
#pragma unroll
    for (int i = 0; i < kGnBatch; ++i)
      if (p + i * a.rpp < t.rows)
        store_pack<E, V>(y + (int64_t)(p + i * a.rpp) * a.C, gn_forward<E, ACT, V, M>(v[i], f, a.thr));
  }
}

// Backward, per tile and channel: sum dz and sum dz xhat.
template <typename E, int ACT, int V, int M>
__global__ void __launch_bounds__(kGnThreads, 3) gn_grad_sums_kernel(GnArgs a) {
  extern __shared__ __align__(16) unsigned char gn_smem[];
  float2* const part = reinterpret_cast<float2*>(gn_smem);  // [rpp][tpr V]
  const GnSpot q = gn_spot(V, a.tpr, a.rpp);
  const GnTile t = gn_tile<V>(a, blockIdx.x, q);
  grid_dependents_may_start();
  if (t.live) {
    GnAffine<V, M> f;
    gn_affine<V, M>(a, t.s, t.c0, &f);
    const int64_t at = (t.s * a.P + t.p0) * a.C + t.c0;
    const E *x = static_cast<const E*>(a.x) + at, *gy = static_cast<const E*>(a.gy) + at;
    float2 acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = make_float2(0.0f, 0.0f);
    for (int p = q.r; p < t.rows; p += kGnGradBatch * a.rpp) {
      Pack<E, V> v[kGnGradBatch], d[kGnGradBatch];
#pragma unroll
      for (int i = 0; i < kGnGradBatch; ++i)
        if (p + i * a.rpp < t.rows) {
          v[i] = load_pack<E, V>(x + (int64_t)(p + i * a.rpp) * a.C);
          d[i] = load_pack<E, V>(gy + (int64_t)(p + i * a.rpp) * a.C);
        }
#pragma unroll
      for (int i = 0; i < kGnGradBatch; ++i)
        if (p + i * a.rpp < t.rows) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            float xc;
            const float dz = gn_dz<E, ACT, V, M>(v[i], d[i], f, j, a.thr, &xc);
            acc[j].x += dz;
            acc[j].y = fmaf(dz, xc, acc[j].y);
          }
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) part[q.r * a.tpr * V + q.cv + j] = make_float2(acc[j].x, acc[j].y * f.rstd[M > 1 ? j : 0]);
  }
  __syncthreads();
  const int width = min(a.tpr * V, a.C - (int)blockIdx.y * a.tpr * V);
  for (int c = threadIdx.x; c < width; c += blockDim.x) {
    float2 v = part[c];
    for (int r = 1; r < a.rpp; ++r) {
      v.x += part[r * a.tpr * V + c].x;
      v.y += part[r * a.tpr * V + c].y;
    }
    *reinterpret_cast<float2*>(a.part + ((int64_t)blockIdx.x * a.C + blockIdx.y * a.tpr * V + c) * 2) = v;
  }
}

// One block per (sample, group): mean(dn) and mean(dn xhat).
__global__ void __launch_bounds__(kGnThreads) gn_grad_finish_kernel(GnArgs a) {
  __shared__ float sm[kGnThreads / 32];
  grid_dependents_may_start();
  grid_wait_for_previous();
  const unsigned u = blockIdx.x, sample = u / (unsigned)a.G;
  const int64_t s = sample, g = u - sample * a.G;
  const float2* part = reinterpret_cast<const float2*>(a.part) + s * a.tiles * a.C + g * a.cg;
  const float* weight = a.weight != nullptr ? a.weight + g * a.cg : nullptr;
  float s1 = 0.0f, s2 = 0.0f;
  gn_each_part(a, [&](int t, int c) {
    const float w = weight != nullptr ? weight[c] : 1.0f;
    const float2 v = part[(int64_t)t * a.C + c];
    s1 = fmaf(w, v.x, s1);
    s2 = fmaf(w, v.y, s2);
  });
  s1 = gn_block_sum<kGnThreads>(s1, sm);
  s2 = gn_block_sum<kGnThreads>(s2, sm);
  if (threadIdx.x == 0) {
    const float inv = 1.0f / ((float)a.P * (float)a.cg);
    a.coef[2 * u] = s1 * inv;
    a.coef[2 * u + 1] = s2 * inv;
  }
}

template <typename E, int ACT, int V, int M>
__global__ void __launch_bounds__(kGnThreads, 3) gn_grad_apply_kernel(GnArgs a) {
  const GnSpot q = gn_spot(V, a.tpr, a.rpp);
  const GnTile t = gn_tile<V>(a, gridDim.x - 1 - (int64_t)blockIdx.x, q);
  grid_dependents_may_start();
  grid_wait_for_previous();
  if (!t.live) return;
  GnAffine<V, M> f;
  gn_affine<V, M>(a, t.s, t.c0, &f);
  float2 k[M];
  gn_groups<V, M>(t.c0, a.cg, [&](int j, int g) {
    if (M > 1 || j == 0)
      k[M > 1 ? j : 0] =
          gn_pull(*reinterpret_cast<const float2*>(a.coef + 2 * (t.s * a.G + g)), f.rstd[M > 1 ? j : 0]);
  });
  const int64_t at = (t.s * a.P + t.p0) * a.C + t.c0;
  const E *x = static_cast<const E*>(a.x) + at, *gy = static_cast<const E*>(a.gy) + at;
  E* dx = static_cast<E*>(a.y) + at;
  for (int p = q.r; p < t.rows; p += kGnGradBatch * a.rpp) {
    Pack<E, V> v[kGnGradBatch], d[kGnGradBatch];
#pragma unroll
    for (int i = 0; i < kGnGradBatch; ++i)
      if (p + i * a.rpp < t.rows) {
        v[i] = load_pack<E, V>(x + (int64_t)(p + i * a.rpp) * a.C);
        d[i] = load_pack<E, V>(gy + (int64_t)(p + i * a.rpp) * a.C);
      }
#pragma unroll
    for (int i = 0; i < kGnGradBatch; ++i)
      if (p + i * a.rpp < t.rows)
        store_pack<E, V>(dx + (int64_t)(p + i * a.rpp) * a.C, gn_backward<E, ACT, V, M>(v[i], d[i], f, k, a.thr));
  }
}

// dweight and dbias: the partial sums over all samples and tiles, in a fixed
// order (the same bits on every run).  32 channels per block, 32 threads each.
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(GnArgs a) {
  __shared__ float2 sm[32][33];
  grid_wait_for_previous();
  const int c = blockIdx.x * 32 + threadIdx.x;
  float2 acc = make_float2(0.0f, 0.0f);
  if (c < a.C) {
#pragma unroll 8
    for (int64_t r = threadIdx.y; r < a.parts; r += 32) {
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

// ---- plans
static int64_t gn_gcd(int64_t a, int64_t b) { return b == 0 ? a : gn_gcd(b, a % b); }

// Channels per thread: 16 bytes of them, else 2, else 1, as shape and pointers allow.
static int gn_vector(size_t eb, int C, const void* x, const void* gy, const void* y) {
  const int wide = 16 / (int)eb;
  for (int v : {wide, 2}) {
    const size_t bytes = v * eb;
    if (C % v == 0 && aligned_to(x, bytes) && aligned_to(gy, bytes) && aligned_to(y, bytes)) return v;
  }
  return 1;
}

// The resident form with k groups and T threads per block in clusters of
// `split`; the shared memory of a block in bytes, 0 when it is above `most`.
static size_t gn_resident_layout(GnArgs* a, int V, int k, int T, int split, bool backward, size_t most) {
  const int64_t width = (int64_t)k * a->cg;
  if (width % V != 0 || width / V > T) return 0;
  a->k = k;
  a->tpr = (int)(width / V);
  a->rpp = T / a->tpr;
  a->threads = T;
  a->split = split;
  a->tiles = (int)ceil_div(a->G, k);
  a->rows = (int)ceil_div(a->P, split);
  a->parts = a->S * split;
  const double held = (double)ceil_div(a->rows, a->rpp) * T * 16 * (backward ? 2 : 1);
  if (held > most) return 0;
  a->held = (int)held;
  const int sets = backward && 32 % a->tpr == 0 ? T / 32 : a->rpp, parts = sets * (int)width;
  const size_t rest = backward ? (size_t)parts + width + 2 * k + T : (size_t)parts / (a->cg % V == 0 ? V : 1) + 2 * k;
  const size_t smem = a->held + rest * sizeof(float2);
  return smem <= most ? smem : 0;
}

// Groups per block, threads and blocks per cluster: rows of at least 64 bytes
// (or whole ones); the fewest blocks per cluster with which three blocks of 256
// threads share an SM, else two of 512; then the most groups that leave enough
// blocks for the GPU.  0: none (the sample is too large, or its rows do not
// divide into packs).  Clusters against tiles, us: forward 16x4096x512 bf16 44
// and 51, 5x3001x320 bf16 11 and 21; backward 16x4096x512 bf16 86 and 86,
// 16x2048x512 fp32 62 and 74, 5x3001x320 bf16 17 and 22.
static size_t gn_resident_plan(GnArgs* a, size_t eb, int V, bool backward) {
  if (V != 16 / (int)eb || a->S >= (1ll << 31) / ((int64_t)a->G * 8)) return 0;
  const int64_t unit = V / gn_gcd(a->cg, V);  // groups that make whole packs
  for (int T : {256, 512}) {
    const size_t most = T == 256 ? 74 * 1024 : 112 * 1024;
    for (int split = 1; split <= 8; split *= 2) {
      int64_t best = 0;
      const int64_t widest = max64((int64_t)T * V / (unit * a->cg), 1);  // a row of packs, one per thread
      for (int64_t n = min64(ceil_div(a->G, unit), widest); n >= 1; --n) {
        const int64_t k = min64(n * unit, a->G);
        if (k < a->G && k * a->cg * (int64_t)eb < 64) break;
        if (gn_resident_layout(a, V, (int)k, T, split, backward, most) == 0) continue;
        best = k;
        if (a->S * a->tiles * split >= 2 * 148) break;
      }
      if (best > 0) return gn_resident_layout(a, V, (int)best, T, split, backward, most);
    }
  }
  return 0;
}

template <typename K>
static cudaError_t gn_launch_resident(K* kernel, const GnArgs& a, size_t smem, cudaStream_t st) {
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid((unsigned)(a.S * a.tiles * a.split)), block((unsigned)a.threads);
  if (a.split > 1) return launch_dependent_cluster(kernel, grid, block, smem, st, (unsigned)a.split, false, a);
  kernel<<<grid, block, smem, st>>>(a);
  return cudaGetLastError();
}

// Tiled form: blocks of up to 256 threads whose rows waste the fewest of them,
// and `per_sm` of them on an SM at once: one wave of tiles where the samples
// divide it, else several of smaller ones; at least 32 positions each (the
// partial sums stay well below the tensor).
static void gn_tiled_rows(int64_t S, int64_t P, int per_sm, int* rows, int* tiles) {
  const int64_t slots = 148 * (int64_t)per_sm;
  const int64_t t = S * 8 <= slots ? slots / max64(S, 1) : ceil_div(4 * slots, S);
  const int64_t r = max64(32, max64(ceil_div(P, t), ceil_div(P, 65535)));
  *rows = (int)min64(r, max64(P, 1));
  *tiles = (int)ceil_div(max64(P, 1), *rows);
}

static void gn_tiled_plan(GnArgs* a, int V, int per_sm) {
  const int per_row = (int)ceil_div(a->C, V);
  a->tpr = per_row > kGnThreads ? kGnThreads : per_row;
  a->rpp = 1;
  a->threads = 32 * (int)ceil_div(a->tpr, 32);
  double best = 0.0;
  for (int rpp = 1; rpp * a->tpr <= kGnThreads && rpp <= 64; ++rpp) {
    const int threads = 32 * (int)ceil_div(rpp * a->tpr, 32);
    const double used = (double)(rpp * a->tpr) / threads * (threads >= 192 ? 1.0 : threads / 192.0);
    if (used > best - 1e-9) {  // of equals the larger
      best = used;
      a->rpp = rpp;
      a->threads = threads;
    }
  }
  gn_tiled_rows(a->S, a->P, per_sm, &a->rows, &a->tiles);
  a->parts = a->S * a->tiles;
}

// Bytes of the partial sums: of the tiled form, and of the resident backward
// pass where that is used.
static size_t gn_part_bytes(size_t eb, int64_t S, int64_t P, int C, int G) {
  int rows, tiles = 0, fewer;
  gn_tiled_rows(S, P, 4, &rows, &tiles);
  gn_tiled_rows(S, P, 3, &rows, &fewer);
  GnArgs a{};
  a.S = S;
  a.P = P;
  a.C = C;
  a.G = G;
  a.cg = C / G;
  const int wide = 16 / (int)eb;
  const int split = C % wide == 0 && gn_resident_plan(&a, eb, wide, true) ? a.split : 1;
  const int most = tiles > fewer ? tiles : fewer;
  return align_up((size_t)S * (most > split ? most : split) * C * 2 * sizeof(float), 256);
}

static int gn_check(int dtype, int64_t S, int64_t P, int C, int G, int act, size_t* eb) {
  SPK_REQUIRE(S >= 0 && P >= 0 && C >= 1 && G >= 1, "invalid shape (S=%lld, P=%lld, C=%d, G=%d)", (long long)S,
              (long long)P, C, G);
  SPK_REQUIRE(C % G == 0, "C=%d is not a multiple of the %d groups", C, G);
  *eb = elem_bytes(dtype);
  SPK_REQUIRE(*eb != 0, "unknown element type %d", dtype);
  SPK_REQUIRE(act == SPK_ACT_NONE || act == SPK_ACT_HEAVISIDE || act == SPK_ACT_SILU,
              "unknown group norm activation %d", act);
  SPK_REQUIRE(C <= (1 << 20) && P < (1ll << 31) && S * G < (1ll << 31) && (P == 0 || S < (1ll << 42) / ((int64_t)C * P)),
              "shape too large (S=%lld, P=%lld, C=%d)", (long long)S, (long long)P, C);
  int rows, tiles;
  gn_tiled_rows(S, P, 4, &rows, &tiles);
  SPK_REQUIRE(S * tiles < (1ll << 31), "too many positions (S=%lld, P=%lld)", (long long)S, (long long)P);
  return SPK_OK;
}

// f(channels per thread, groups among them at most)
template <typename E, typename F>
inline void with_gn_vector(int V, int cg, F&& f) {
  constexpr int kWide = 16 / (int)sizeof(E);
  if (V == kWide && cg % kWide == 0)
    f(std::integral_constant<int, kWide>{}, std::integral_constant<int, 1>{});
  else if (V == kWide)
    f(std::integral_constant<int, kWide>{}, std::integral_constant<int, kWide>{});
  else if (V == 2)
    f(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
  else
    f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
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

extern "C" size_t spk_group_norm_workspace_bytes(int dtype, int64_t S, int64_t P, int C, int G) {
  const size_t eb = spk::elem_bytes(dtype);
  if (eb == 0 || S <= 0 || P <= 0 || C <= 0 || G <= 0 || C % G != 0) return 0;
  return spk::gn_part_bytes(eb, S, P, C, G) + (size_t)S * G * 2 * sizeof(float);
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
  if (workspace == nullptr || workspace_bytes < spk_group_norm_workspace_bytes(dtype, S, P, C, G))
    return spk::fail(SPK_EWORKSPACE, "group norm needs a workspace of %zu bytes",
                     spk_group_norm_workspace_bytes(dtype, S, P, C, G));
  SPK_REQUIRE(spk::aligned_to(workspace, 16), "the workspace must be 16-byte aligned");
  spk::GnArgs a{};
  a.x = X;
  a.weight = weight;
  a.bias = bias;
  a.y = Y;
  a.part = static_cast<float*>(workspace);
  float* tail = reinterpret_cast<float*>(static_cast<char*>(workspace) + spk::gn_part_bytes(eb, S, P, C, G));
  a.mean = mean != nullptr ? mean : tail;
  a.rstd = rstd != nullptr ? rstd : tail + S * G;
  a.S = S;
  a.P = P;
  a.C = C;
  a.G = G;
  a.cg = C / G;
  a.eps = eps;
  a.thr = thr;
  cudaStream_t st = (cudaStream_t)stream;
  const int V = spk::gn_vector(eb, C, X, nullptr, Y);
  if (const size_t held = spk::gn_resident_plan(&a, eb, V, false)) {
    cudaError_t rc = cudaSuccess;
    a.mean = mean;
    a.rstd = rstd;
    spk::with_elem(dtype, [&](auto e) {
      using E = decltype(e);
      spk::with_gn_act(act, [&](auto ac) {
        constexpr int ACT = decltype(ac)::value;
        rc = a.cg % V == 0 ? spk::gn_launch_resident(spk::gn_resident_kernel<E, ACT, true>, a, held, st)
                           : spk::gn_launch_resident(spk::gn_resident_kernel<E, ACT, false>, a, held, st);
      });
    });
    SPK_CUDA_TRY(rc);
    spk::count_launch(1);
    return SPK_OK;
  }
  spk::gn_tiled_plan(&a, V, 4);
  // a kernel that starts while the one before it drains
  cudaError_t rc = cudaSuccess;
  auto launch = [&](auto kernel, dim3 grid, dim3 block) {
    const cudaError_t e = spk::launch_dependent(kernel, grid, block, 0, st, a);
    if (rc == cudaSuccess) rc = e;
  };
  const dim3 grid((unsigned)a.parts, (unsigned)spk::ceil_div(C, a.tpr * V)), block((unsigned)a.threads);
  const size_t smem = (size_t)a.rpp * a.tpr * V * sizeof(float2);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    spk::with_gn_vector<E>(V, a.cg, [&](auto vc, auto mc) {
      constexpr int VV = decltype(vc)::value, MM = decltype(mc)::value;
      spk::gn_stats_kernel<E, VV><<<grid, block, smem, st>>>(a);
      launch(spk::gn_stats_finish_kernel, dim3((unsigned)(S * G)), dim3(spk::kGnThreads));
      spk::with_gn_act(act, [&](auto ac) {
        launch(spk::gn_apply_kernel<E, decltype(ac)::value, VV, MM>, grid, block);
      });
    });
  });
  SPK_CUDA_TRY(rc);
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
  if (workspace == nullptr || workspace_bytes < spk_group_norm_workspace_bytes(dtype, S, P, C, G))
    return spk::fail(SPK_EWORKSPACE, "group norm needs a workspace of %zu bytes",
                     spk_group_norm_workspace_bytes(dtype, S, P, C, G));
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
  a.coef = reinterpret_cast<float*>(static_cast<char*>(workspace) + spk::gn_part_bytes(eb, S, P, C, G));
  a.dweight = dweight;
  a.dbias = dbias;
  a.S = S;
  a.P = P;
  a.C = C;
  a.G = G;
  a.cg = C / G;
  a.thr = thr;
  const int V = spk::gn_vector(eb, C, X, GY, DX);
  const bool params = dweight != nullptr || dbias != nullptr;
  // a kernel that starts while the one before it drains
  cudaError_t rc = cudaSuccess;
  auto launch = [&](auto kernel, dim3 grid, dim3 block) {
    const cudaError_t e = spk::launch_dependent(kernel, grid, block, 0, st, a);
    if (rc == cudaSuccess) rc = e;
  };
  if (const size_t held = spk::gn_resident_plan(&a, eb, V, true)) {
    if (!params) a.part = nullptr;
    spk::with_elem(dtype, [&](auto e) {
      using E = decltype(e);
      spk::with_gn_act(act, [&](auto ac) {
        constexpr int ACT = decltype(ac)::value;
        rc = a.cg % V == 0 ? spk::gn_launch_resident(spk::gn_resident_backward_kernel<E, ACT, true>, a, held, st)
                           : spk::gn_launch_resident(spk::gn_resident_backward_kernel<E, ACT, false>, a, held, st);
      });
    });
    SPK_CUDA_TRY(rc);
    spk::count_launch(1);
  } else {
    spk::gn_tiled_plan(&a, V, 3);
    const dim3 grid((unsigned)a.parts, (unsigned)spk::ceil_div(C, a.tpr * V)), block((unsigned)a.threads);
    const size_t smem = (size_t)a.rpp * a.tpr * V * sizeof(float2);
    spk::with_elem(dtype, [&](auto e) {
      using E = decltype(e);
      spk::with_gn_vector<E>(V, a.cg, [&](auto vc, auto mc) {
        constexpr int VV = decltype(vc)::value, MM = decltype(mc)::value;
        spk::with_gn_act(act, [&](auto ac) {
          constexpr int ACT = decltype(ac)::value;
          spk::gn_grad_sums_kernel<E, ACT, VV, MM><<<grid, block, smem, st>>>(a);
          launch(spk::gn_grad_finish_kernel, dim3((unsigned)(S * G)), dim3(spk::kGnThreads));
          launch(spk::gn_grad_apply_kernel<E, ACT, VV, MM>, grid, block);
        });
      });
    });
    spk::count_launch(3);
  }
  if (params) {
    launch(spk::gn_param_grad_kernel, dim3((unsigned)spk::ceil_div(C, 32)), dim3(32, 32));
    spk::count_launch(1);
  }
  SPK_CUDA_TRY(rc);
  SPK_LAUNCH_CHECK();
  return SPK_OK;
}
