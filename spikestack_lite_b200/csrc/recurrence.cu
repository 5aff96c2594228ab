// Gated linear recurrence over time and its backward pass.  Per batch row b
// and channel d, over the steps t = 0 .. len_b - 1:
//   gate form:   h_t = a_t h_{t-1} + x_t                      (a_t given)
//   leaky form:  h_t = h_{t-1} + q_t (x_t - h_{t-1}),          q_t = 1 - a_t,
//                a_t = sigmoid(gate_t)
// with h_{-1} the initial state.  Backward, with g_t the
// gradient of h_t:
//   g_t = gh_t + a_{t+1} g_{t+1}   (the last state's gradient enters behind len_b - 1)
//   gate form:   dx_t = g_t,       dgate_t = g_t h_{t-1}
//   leaky form:  dx_t = q_t g_t,   dgate_t = g_t (h_{t-1} - x_t) a_t q_t
// and dstate = a_0 g_0.  States and sums are fp32 whatever the element type.
#include "elem.cuh"

namespace spk {

struct RecArgs {
  const void* x;
  const void* gate;
  const void* gh;         // backward: gradient of h, or null
  const float* h0;        // [B, D] or null
  const float* glast;     // backward: gradient of the last state [B, D], or null
  const int32_t* lengths; // [B] or null
  void* h;
  float* last;            // [B, D]
  float* carry;           // [chunks - 1, B, D]: the state before steps 64, 128, ...; or null
  void* dx;
  void* dgate;
  float* dh0;
  int64_t B, L, D;
  int64_t x_b, x_t, g_b, g_t, h_b, h_t, o_b, o_t;  // strides in elements (h: h or gh; o: dx and dgate)
};

// The decay of one or more steps as one float per form: `coeff` from the gate,
// `step` the new state, `apply` A h + H for a joined decay A, `join` the decay
// of two in a row, `back` the gradient that passes a step, dx and dgate the
// gradients of its inputs (dgate from grad_base of the state before and x).
// kept_gate is the gate, kept the decay, of a step that keeps the state.
struct GateForm {
  __device__ static float kept_gate() { return 1.0f; }
  __device__ static float kept() { return 1.0f; }
  __device__ static float coeff(float gate) { return gate; }
  __device__ static float step(float h, float a, float x) { return fmaf(a, h, x); }
  __device__ static float apply(float a, float h, float H) { return fmaf(a, h, H); }
  __device__ static float join(float a, float b) { return a * b; }
  __device__ static float back(float g, float a) { return a * g; }
  __device__ static float dx(float g, float) { return g; }
  __device__ static float grad_base(float h, float) { return h; }
  __device__ static float dgate(float g, float, float base) { return g * base; }
};

// Leaky form: whichever of a and q = 1 - a is at most one half, its sign bit
// set when it is a.  Both ends of the gate keep their relative accuracy: a
// slow channel's q and a fast channel's a are never differences from 1, and
// neither are those of joined steps.
struct LeakyForm {
  __device__ static float kept_gate() { return __int_as_float(0x7f800000); }  // q = 0
  __device__ static float kept() { return 0.0f; }
  __device__ static float coeff(float gate) {
    const float e = expf(-fabsf(gate));
    return copysignf(__fdividef(e, 1.0f + e), gate);
  }
  __device__ static bool is_a(float c) { return __float_as_int(c) < 0; }
  __device__ static float step(float h, float c, float x) {
    const bool fast = is_a(c);  // x + a (h - x), else h + q (x - h)
    const float base = fast ? x : h;
    return fmaf(fabsf(c), (fast ? h : x) - base, base);
  }
  __device__ static float apply(float c, float h, float H) {
    return is_a(c) ? fmaf(-c, h, H) : fmaf(-c, h, h) + H;
  }
  __device__ static float join(float c, float d) {
    if (!is_a(c) && !is_a(d)) {
      const float q = fmaf(-c, d, c) + d;  // 1 - (1 - c)(1 - d), at most 3/4
      return q <= 0.5f ? q : q - 1.0f;
    }
    return -((is_a(c) ? -c : 1.0f - c) * (is_a(d) ? -d : 1.0f - d));
  }
  __device__ static float back(float g, float c) { return is_a(c) ? -c * g : fmaf(-c, g, g); }
  __device__ static float dx(float g, float c) { return is_a(c) ? fmaf(c, g, g) : c * g; }
  __device__ static float grad_base(float h, float x) { return h - x; }
  __device__ static float dgate(float g, float c, float base) {
    const float s = fabsf(c);
    return g * base * fmaf(-s, s, s);
  }
};

__device__ __forceinline__ int64_t rec_len(const RecArgs& a, int64_t b) {
  if (a.lengths == nullptr) return a.L;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : (n > a.L ? a.L : n);
}

// ---- tiles
// A tile is up to 64 steps of 128 neighbouring channels of one batch row (one
// "chain" of tiles along time).  A warp holds 8 steps of it in registers, a
// lane 4 channels; a block is 8 warps, `wt` of them along time (8 when there
// are more than 32 steps) and 8 / wt along chains.  Each warp reduces its
// steps to one affine map h -> A h + H, the warps' maps meet in shared memory,
// and every warp then runs its steps once more from its own start, in the
// order of the definition.
//
// More than 64 steps: the tiles of a chain are joined in the same launch.  A
// block takes the next tile in time-major order (a ticket, so every tile it
// may wait for has been taken already), publishes its map, looks back over its
// predecessors' maps to the nearest finished state, and publishes the state
// behind itself: x and gate are read once however few chains there are.
constexpr int kRecSteps = 8;                      // steps per warp
constexpr int kRecWarps = 8;                      // warps per block
constexpr int kRecCols = 128;                     // channels per warp: 4 per lane
constexpr int kRecChunk = kRecSteps * kRecWarps;  // steps per tile, and between the states kept for the backward pass

struct RecPlan {
  int64_t chains, groups;  // chains = B * groups of 128 channels
  int64_t tiles;           // blocks
  int chunks, wt;
  uint32_t* ticket;        // followed by one flag per tile; null with one chunk
  float* maps;             // [tiles][2][128]: A, H
  float* states;           // [tiles][128]: the state behind the tile
};

struct Quad {
  float v[4];
};

// The lane's 4 channels of `n` (at most 128) starting at p: neighbours with
// one access (ALIGNED), or every 32nd.
template <bool ALIGNED>
__device__ __forceinline__ int rec_col(int lane, int i) {
  return ALIGNED ? 4 * lane + i : lane + 32 * i;
}

template <bool ALIGNED, typename E>
__device__ __forceinline__ Quad rec_load(const E* p, int lane, int n, float other) {
  Quad q;
  if (ALIGNED) {
    if (4 * lane < n) {
      const Pack<E, 4> e = load_pack<E, 4>(p + 4 * lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) q.v[i] = elem_to_f32(e.e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) q.v[i] = other;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = lane + 32 * i < n ? elem_to_f32(p[lane + 32 * i]) : other;
  }
  return q;
}

template <bool ALIGNED, typename E>
__device__ __forceinline__ void rec_store(E* p, int lane, int n, const Quad& q) {
  if (ALIGNED) {
    if (4 * lane < n) {
      Pack<E, 4> e;
#pragma unroll
      for (int i = 0; i < 4; ++i) e.e[i] = elem_from_f32<E>(q.v[i]);
      store_pack<E, 4>(p + 4 * lane, e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < n) p[lane + 32 * i] = elem_from_f32<E>(q.v[i]);
  }
}

__device__ __forceinline__ void st_flag(uint32_t* p, uint32_t v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_flag(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ Quad quad_cg(const float* p) {
  const float4 f = __ldcg(reinterpret_cast<const float4*>(p));
  return Quad{{f.x, f.y, f.z, f.w}};
}
__device__ __forceinline__ void quad_st(float* p, const Quad& q) {
  *reinterpret_cast<float4*>(p) = make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
}

constexpr uint32_t kRecMap = 1, kRecState = 2;  // flag of a tile: its map, then the state behind it, is published

// The state entering a tile, by one warp: walks back over the tiles at
// tile - chains, tile - 2 chains, ... (`before` of them) to the nearest
// published state, or to `first`, the state in front of them all, waiting for
// the maps of the tiles between; then applies these maps in time order.  Every
// state is the map of its tile applied to the state before, wherever the walk
// ended, so the result does not depend on the order in which tiles finished.
template <typename Form>
__device__ __forceinline__ Quad rec_look_back(const RecPlan& p, int64_t tile, int before, const Quad& first, int lane) {
  const uint32_t* flags = p.ticket + 1;
  int found = before;  // tiles between this one and the state
  for (int base = 0; base < before; base += 32) {
    const int k = base + lane;  // lane l looks at the l-th tile back of this round
    uint32_t f = kRecState;     // in front of the first tile: `first`
    int nearest;
    uint64_t t_start = 0;
    for (int polls = 0;; ++polls) {
      if (k < before) f = ld_flag(flags + (tile - (int64_t)(k + 1) * p.chains));
      const uint32_t states = __ballot_sync(0xffffffffu, f == kRecState);
      const uint32_t open = __ballot_sync(0xffffffffu, f == 0);
      nearest = states ? __ffs(states) - 1 : 32;
      const uint32_t needed = nearest >= 32 ? 0xffffffffu : (1u << nearest) - 1u;
      if ((open & needed) == 0) break;
      if (polls == 0) t_start = global_ns();
      const bool late = (polls & 63) == 63 && global_ns() - t_start > kSpinLimitNs;
      if (__any_sync(0xffffffffu, late)) {  // a predecessor never published: report, and leave with a wrong state
        if (lane == 0) report_device_error(SPK_DEV_SCAN_TIMEOUT);
        return first;
      }
    }
    if (nearest < 32) {
      found = base + nearest;
      break;
    }
  }
  __syncwarp();
  Quad s = found < before ? quad_cg(p.states + (tile - (int64_t)(found + 1) * p.chains) * kRecCols + 4 * lane) : first;
#pragma unroll 4
  for (int j = found; j > 0; --j) {
    const float* m = p.maps + (tile - (int64_t)j * p.chains) * 2 * kRecCols + 4 * lane;
    const Quad A = quad_cg(m), H = quad_cg(m + kRecCols);
#pragma unroll
    for (int i = 0; i < 4; ++i) s.v[i] = Form::apply(A.v[i], s.v[i], H.v[i]);
  }
  return s;
}

// Publishes one warp's worth of data (the lanes' quads, already stored) of a tile.
__device__ __forceinline__ void rec_publish(const RecPlan& p, int64_t tile, uint32_t what, int lane) {
  __threadfence();
  __syncwarp();
  if (lane == 0) st_flag(p.ticket + 1 + tile, what);
}

// One warp's part of joining a tile: publishes the tile's map (of the warps'
// maps sA, sH, in time order or in reverse), looks back, publishes the state
// behind the tile (unless it is the last of its chain) and returns the one
// in front of it.
template <typename Form>
__device__ __forceinline__ Quad rec_join(const RecPlan& p, int64_t tile, int before, const Quad& first,
                                         const float (*sA)[kRecCols], const float (*sH)[kRecCols], bool reverse,
                                         int lane, Quad* behind) {
  const bool more = before + 1 < p.chunks;
  Quad A, H;
  if (more) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      A.v[i] = Form::kept();
      H.v[i] = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kRecWarps; ++k) {
      const int w = reverse ? kRecWarps - 1 - k : k;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        H.v[i] = Form::apply(sA[w][4 * lane + i], H.v[i], sH[w][4 * lane + i]);
        A.v[i] = Form::join(A.v[i], sA[w][4 * lane + i]);
      }
    }
    if (before > 0) {
      float* m = p.maps + tile * 2 * kRecCols + 4 * lane;
      quad_st(m, A);
      quad_st(m + kRecCols, H);
      rec_publish(p, tile, kRecMap, lane);
    }
  }
  const Quad s = before > 0 ? rec_look_back<Form>(p, tile, before, first, lane) : first;
  if (more) {
#pragma unroll
    for (int i = 0; i < 4; ++i) behind->v[i] = Form::apply(A.v[i], s.v[i], H.v[i]);
    quad_st(p.states + tile * kRecCols + 4 * lane, *behind);
    rec_publish(p, tile, kRecState, lane);
  }
  return s;
}

// The block's tile: the chunk (time) and chain of this warp; false past the end.
template <bool SPLIT>
__device__ __forceinline__ bool rec_tile(const RecPlan& p, int warp, int64_t* tile, int* chunk, int64_t* chain) {
  if (SPLIT) {
    __shared__ uint32_t s_ticket;
    if (threadIdx.x == 0) s_ticket = atomicAdd(p.ticket, 1u);
    __syncthreads();
    *tile = s_ticket;
    *chunk = (int)(*tile / p.chains);
    *chain = *tile - (int64_t)*chunk * p.chains;
    return true;
  }
  *tile = blockIdx.x;
  *chunk = 0;
  *chain = (int64_t)blockIdx.x * (kRecWarps / p.wt) + warp / p.wt;
  return *chain < p.chains;
}

template <typename E, typename Form, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(32 * kRecWarps, 2) recurrence_kernel(RecArgs a, RecPlan p) {
  __shared__ float sA[kRecWarps][kRecCols], sH[kRecWarps][kRecCols], sC[kRecCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t tile, chain;
  int chunk;
  const bool live = rec_tile<SPLIT>(p, warp, &tile, &chunk, &chain);
  const int wt = SPLIT ? kRecWarps : p.wt, w = SPLIT ? warp : warp % wt;
  const int64_t b = live ? chain / p.groups : 0, col = live ? (chain - b * p.groups) * kRecCols : 0;
  const int n = live ? (int)min64(a.D - col, kRecCols) : 0;
  const int64_t t0 = (int64_t)chunk * kRecChunk + w * kRecSteps;
  const int64_t len = live ? rec_len(a, b) : 0;
  const E* x = static_cast<const E*>(a.x) + b * a.x_b + t0 * a.x_t + col;
  const E* gate = static_cast<const E*>(a.gate) + b * a.g_b + t0 * a.g_t + col;
  Quad c[kRecSteps], u[kRecSteps];
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {  // a step behind the end keeps the state
    const int m = t0 + j < len ? n : 0;
    c[j] = rec_load<ALIGNED>(gate + j * a.g_t, lane, m, Form::kept_gate());
    u[j] = rec_load<ALIGNED>(x + j * a.x_t, lane, m, 0.0f);
  }
  Quad h = {{0.0f, 0.0f, 0.0f, 0.0f}};
  if (!SPLIT && a.h0 != nullptr) h = rec_load<ALIGNED>(a.h0 + b * a.D + col, lane, n, 0.0f);
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j].v[i] = Form::coeff(c[j].v[i]);
  if (SPLIT || wt > 1) {
    Quad A, H;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      A.v[i] = c[0].v[i];
      H.v[i] = Form::step(0.0f, c[0].v[i], u[0].v[i]);
    }
#pragma unroll
    for (int j = 1; j < kRecSteps; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        H.v[i] = Form::step(H.v[i], c[j].v[i], u[j].v[i]);
        A.v[i] = Form::join(A.v[i], c[j].v[i]);
      }
    quad_st(&sA[warp][4 * lane], A);
    quad_st(&sH[warp][4 * lane], H);
    __syncthreads();
    if (SPLIT) {
      if (warp == 0) {
        Quad first = {{0.0f, 0.0f, 0.0f, 0.0f}}, behind;
        if (a.h0 != nullptr) first = rec_load<ALIGNED>(a.h0 + b * a.D + col, lane, n, 0.0f);
        quad_st(&sC[4 * lane], rec_join<Form>(p, tile, chunk, first, sA, sH, false, lane, &behind));
        if (chunk + 1 < p.chunks && a.carry != nullptr)
          rec_store<ALIGNED>(a.carry + ((int64_t)chunk * a.B + b) * a.D + col, lane, n, behind);
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) h.v[i] = sC[4 * lane + i];
    }
    for (int k = warp - w; k < warp; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) h.v[i] = Form::apply(sA[k][4 * lane + i], h.v[i], sH[k][4 * lane + i]);
  }
  if (!live) return;
  E* out = static_cast<E*>(a.h) + b * a.h_b + t0 * a.h_t + col;
  const Quad zero = {{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {
#pragma unroll
    for (int i = 0; i < 4; ++i) h.v[i] = Form::step(h.v[i], c[j].v[i], u[j].v[i]);
    if (t0 + j < a.L) rec_store<ALIGNED>(out + j * a.h_t, lane, n, t0 + j < len ? h : zero);
  }
  if (chunk + 1 == p.chunks && w + 1 == wt) rec_store<ALIGNED>(a.last + b * a.D + col, lane, n, h);
}

// Backward: the same tiles, taken from the end.  A tile runs its steps forward
// from the state the forward pass kept (h is not read back from memory, where
// it was rounded), and backwards from the gradient that reaches it, whose
// affine map has the same decay.
template <typename E, typename Form, bool ALIGNED, bool SPLIT>
__global__ void __launch_bounds__(32 * kRecWarps, 2) recurrence_backward_kernel(RecArgs a, RecPlan p) {
  __shared__ float sA[kRecWarps][kRecCols], sH[kRecWarps][kRecCols], sG[kRecWarps][kRecCols], sC[kRecCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t tile, chain;
  int back;
  const bool live = rec_tile<SPLIT>(p, warp, &tile, &back, &chain);
  const int chunk = p.chunks - 1 - back;
  const int wt = SPLIT ? kRecWarps : p.wt, w = SPLIT ? warp : warp % wt;
  const int64_t b = live ? chain / p.groups : 0, col = live ? (chain - b * p.groups) * kRecCols : 0;
  const int n = live ? (int)min64(a.D - col, kRecCols) : 0;
  const int64_t t0 = (int64_t)chunk * kRecChunk + w * kRecSteps;
  const int64_t len = live ? rec_len(a, b) : 0;
  const E* x = static_cast<const E*>(a.x) + b * a.x_b + t0 * a.x_t + col;
  const E* gate = static_cast<const E*>(a.gate) + b * a.g_b + t0 * a.g_t + col;
  const E* gh = static_cast<const E*>(a.gh) + b * a.h_b + t0 * a.h_t + col;
  const Quad zero = {{0.0f, 0.0f, 0.0f, 0.0f}};
  Quad c[kRecSteps], u[kRecSteps], g[kRecSteps];
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j) {
    const int m = t0 + j < len ? n : 0;
    c[j] = rec_load<ALIGNED>(gate + j * a.g_t, lane, m, Form::kept_gate());
    u[j] = rec_load<ALIGNED>(x + j * a.x_t, lane, m, 0.0f);
    g[j] = rec_load<ALIGNED>(gh + j * a.h_t, lane, a.gh != nullptr ? m : 0, 0.0f);
  }
  Quad h = zero, later = zero;
  if (live) {
    const float* start = chunk > 0 ? a.carry + ((int64_t)(chunk - 1) * a.B + b) * a.D + col
                                   : (a.h0 != nullptr ? a.h0 + b * a.D + col : nullptr);
    if (start != nullptr) h = rec_load<ALIGNED>(start, lane, n, 0.0f);
    if (a.glast != nullptr && (!SPLIT || warp == 0)) later = rec_load<ALIGNED>(a.glast + b * a.D + col, lane, n, 0.0f);
  }
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) c[j].v[i] = Form::coeff(c[j].v[i]);
  if (SPLIT || wt > 1) {
    Quad A, H, G;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      A.v[i] = c[0].v[i];
      H.v[i] = Form::step(0.0f, c[0].v[i], u[0].v[i]);
      G.v[i] = 0.0f;
    }
#pragma unroll
    for (int j = 1; j < kRecSteps; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        H.v[i] = Form::step(H.v[i], c[j].v[i], u[j].v[i]);
        A.v[i] = Form::join(A.v[i], c[j].v[i]);
      }
#pragma unroll
    for (int j = kRecSteps - 1; j >= 0; --j)
#pragma unroll
      for (int i = 0; i < 4; ++i) G.v[i] = Form::back(g[j].v[i] + G.v[i], c[j].v[i]);
    quad_st(&sA[warp][4 * lane], A);
    quad_st(&sH[warp][4 * lane], H);
    quad_st(&sG[warp][4 * lane], G);
    __syncthreads();
    if (SPLIT) {
      if (warp == 0) {
        Quad behind;
        quad_st(&sC[4 * lane], rec_join<Form>(p, tile, back, later, sA, sG, true, lane, &behind));
      }
    }
    for (int k = warp - w; k < warp; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) h.v[i] = Form::apply(sA[k][4 * lane + i], h.v[i], sH[k][4 * lane + i]);
  }
  // forward once more; what dgate needs of the state takes x's place
#pragma unroll
  for (int j = 0; j < kRecSteps; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float before = h.v[i];
      h.v[i] = Form::step(before, c[j].v[i], u[j].v[i]);
      u[j].v[i] = Form::grad_base(before, u[j].v[i]);
    }
  if (SPLIT || wt > 1) {
    if (SPLIT) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) later.v[i] = sC[4 * lane + i];
    }
    for (int k = warp - w + wt - 1; k > warp; --k)
#pragma unroll
      for (int i = 0; i < 4; ++i) later.v[i] = Form::apply(sA[k][4 * lane + i], later.v[i], sG[k][4 * lane + i]);
  }
  if (!live) return;
  E* dx = static_cast<E*>(a.dx) + b * a.o_b + t0 * a.o_t + col;
  E* dg = static_cast<E*>(a.dgate) + b * a.o_b + t0 * a.o_t + col;
#pragma unroll
  for (int j = kRecSteps - 1; j >= 0; --j) {
    Quad ox, og;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float total = g[j].v[i] + later.v[i];
      ox.v[i] = Form::dx(total, c[j].v[i]);
      og.v[i] = Form::dgate(total, c[j].v[i], u[j].v[i]);
      later.v[i] = Form::back(total, c[j].v[i]);
    }
    if (t0 + j < a.L) {
      const bool on = t0 + j < len;
      rec_store<ALIGNED>(dx + j * a.o_t, lane, n, on ? ox : zero);
      rec_store<ALIGNED>(dg + j * a.o_t, lane, n, on ? og : zero);
    }
  }
  if (a.dh0 != nullptr && chunk == 0 && w == 0) rec_store<ALIGNED>(a.dh0 + b * a.D + col, lane, n, later);
}

// One step of the recurrence over n cells: out (element type) and the new
// state (fp32; may be the old state's own buffer).
template <typename E, typename Form>
__global__ void __launch_bounds__(256) recurrence_step_kernel(const E* __restrict__ x, const E* __restrict__ gate,
                                                              const float* state, int64_t n, E* __restrict__ out,
                                                              float* new_state) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const float h = Form::step(state[i], Form::coeff(elem_to_f32(gate[i])), elem_to_f32(x[i]));
  out[i] = elem_from_f32<E>(h);
  new_state[i] = h;
}

template <typename F>
inline bool with_form(int form, F&& f) {
  if (form == SPK_REC_GATE) {
    f(GateForm{});
    return true;
  }
  if (form == SPK_REC_LEAKY) {
    f(LeakyForm{});
    return true;
  }
  return false;
}

// Shape, type and alignment checks shared by the recurrence's entry points.
static int rec_check(int dtype, int form, int64_t B, int64_t L, int64_t D, size_t* eb) {
  SPK_REQUIRE(B >= 0 && L >= 0 && D >= 0, "invalid shape (B=%lld, L=%lld, D=%lld)", (long long)B, (long long)L,
              (long long)D);
  *eb = elem_bytes(dtype);
  SPK_REQUIRE(*eb != 0, "unknown element type %d", dtype);
  SPK_REQUIRE(form == SPK_REC_GATE || form == SPK_REC_LEAKY, "unknown recurrence form %d", form);
  SPK_REQUIRE(L < (1ll << 31) && D < (1ll << 31) && (D == 0 || B < (1ll << 37) / D),
              "shape too large (B=%lld, L=%lld, D=%lld)", (long long)B, (long long)L, (long long)D);
  SPK_REQUIRE((double)B * ceil_div(D, kRecCols) * max64(ceil_div(L, kRecChunk), 1) < 2147483647.0,
              "too many steps and channels (B=%lld, L=%lld, D=%lld)", (long long)B, (long long)L, (long long)D);
  return SPK_OK;
}

static bool rec_aligned(const void* p, size_t eb, int64_t stride_b, int64_t stride_t) {
  return aligned_to(p, 4 * eb) && stride_b % 4 == 0 && stride_t % 4 == 0;
}

// Fills the plan from the workspace; batch rows that follow one another like
// channels (no lengths, batch stride D everywhere) become channels first, so
// that narrow rows share a warp.
static void rec_plan(RecArgs* a, RecPlan* p, bool merge, void* workspace) {
  if (merge && a->lengths == nullptr) {
    a->D *= a->B;
    a->B = 1;
  }
  p->groups = ceil_div(a->D, kRecCols);
  p->chains = a->B * p->groups;
  p->chunks = (int)max64(ceil_div(a->L, kRecChunk), 1);
  p->wt = 1;
  while (p->wt < kRecWarps && (int64_t)p->wt * kRecSteps < a->L) p->wt *= 2;
  p->tiles = p->chunks > 1 ? p->chains * p->chunks : ceil_div(p->chains, kRecWarps / p->wt);
  if (p->chunks > 1) {
    p->ticket = static_cast<uint32_t*>(workspace);
    p->maps = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up(4 * (size_t)(p->tiles + 1), 256));
    p->states = p->maps + p->tiles * 2 * kRecCols;
  }
}

static int rec_workspace_check(int64_t B, int64_t L, int64_t D, const void* workspace, size_t bytes) {
  const size_t need = spk_recurrence_workspace_bytes(B, L, D);
  if (need > 0 && (workspace == nullptr || bytes < need))
    return fail(SPK_EWORKSPACE, "the recurrence needs a workspace of %zu bytes", need);
  SPK_REQUIRE(aligned_to(workspace, 16), "the workspace must be 16-byte aligned");
  return SPK_OK;
}

// The kernel of a plan, its counters cleared first when tiles are joined.
#define SPK_REC_LAUNCH(KERNEL)                                                                              \
  if (p.chunks > 1)                                                                                         \
    SPK_CUDA_TRY(cudaMemsetAsync(p.ticket, 0, 4 * (size_t)(p.tiles + 1), st));                              \
  spk::with_elem(dtype, [&](auto e) {                                                                       \
    spk::with_form(form, [&](auto f) {                                                                      \
      using E = decltype(e);                                                                                \
      using F = decltype(f);                                                                                \
      const dim3 grid((unsigned)p.tiles), block(32 * spk::kRecWarps);                                       \
      if (p.chunks > 1 && aligned)                                                                          \
        spk::KERNEL<E, F, true, true><<<grid, block, 0, st>>>(a, p);                                        \
      else if (p.chunks > 1)                                                                                \
        spk::KERNEL<E, F, false, true><<<grid, block, 0, st>>>(a, p);                                       \
      else if (aligned)                                                                                     \
        spk::KERNEL<E, F, true, false><<<grid, block, 0, st>>>(a, p);                                       \
      else                                                                                                  \
        spk::KERNEL<E, F, false, false><<<grid, block, 0, st>>>(a, p);                                      \
    });                                                                                                     \
  });                                                                                                       \
  SPK_LAUNCH_CHECK();                                                                                       \
  spk::count_launch(1)

}  // namespace spk

extern "C" int spk_recurrence_chunk(void) { return spk::kRecChunk; }

extern "C" size_t spk_recurrence_workspace_bytes(int64_t B, int64_t L, int64_t D) {
  if (B <= 0 || D <= 0 || L <= spk::kRecChunk) return 0;
  const size_t tiles = (size_t)(B * spk::ceil_div(D, spk::kRecCols) * spk::ceil_div(L, spk::kRecChunk));
  return spk::align_up(4 * (tiles + 1), 256) + tiles * 3 * spk::kRecCols * sizeof(float);
}

extern "C" int spk_recurrence(const void* x, int64_t x_stride_b, int64_t x_stride_t, const void* gate,
                              int64_t g_stride_b, int64_t g_stride_t, int dtype, int form, int64_t B, int64_t L,
                              int64_t D, const float* state, const int32_t* lengths, void* h, int64_t h_stride_b,
                              int64_t h_stride_t, float* last, float* carry, void* workspace, size_t workspace_bytes,
                              spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, B, L, D, &eb)) return rc;
  if (B == 0 || D == 0) return SPK_OK;
  SPK_REQUIRE(last != nullptr && (L == 0 || (x != nullptr && gate != nullptr && h != nullptr)),
              "x, gate, h and last must be non-null");
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(h, eb) &&
                  spk::aligned_to(state, 4) && spk::aligned_to(lengths, 4) && spk::aligned_to(last, 4) &&
                  spk::aligned_to(carry, 4),
              "tensors must be aligned to their elements");
  if (int rc = spk::rec_workspace_check(B, L, D, workspace, workspace_bytes)) return rc;
  spk::RecArgs a{};
  a.x = x;
  a.gate = gate;
  a.h0 = state;
  a.lengths = lengths;
  a.h = h;
  a.last = last;
  a.carry = carry;
  a.B = B;
  a.L = L;
  a.D = D;
  a.x_b = x_stride_b;
  a.x_t = x_stride_t;
  a.g_b = g_stride_b;
  a.g_t = g_stride_t;
  a.h_b = h_stride_b;
  a.h_t = h_stride_t;
  const bool aligned = D % 4 == 0 && spk::rec_aligned(x, eb, x_stride_b, x_stride_t) &&
                       spk::rec_aligned(gate, eb, g_stride_b, g_stride_t) &&
                       spk::rec_aligned(h, eb, h_stride_b, h_stride_t) && spk::aligned_to(state, 16) &&
                       spk::aligned_to(last, 16) && spk::aligned_to(carry, 16);
  cudaStream_t st = (cudaStream_t)stream;
  spk::RecPlan p{};
  spk::rec_plan(&a, &p, x_stride_b == D && g_stride_b == D && h_stride_b == D, workspace);
  SPK_REC_LAUNCH(recurrence_kernel);
  return SPK_OK;
}

extern "C" int spk_recurrence_backward(const void* x, int64_t x_stride_b, int64_t x_stride_t, const void* gate,
                                       int64_t g_stride_b, int64_t g_stride_t, const void* gh, int64_t gh_stride_b,
                                       int64_t gh_stride_t, int dtype, int form, int64_t B, int64_t L, int64_t D,
                                       const float* state, const int32_t* lengths, const float* carry,
                                       const float* glast, void* dx, void* dgate, int64_t d_stride_b,
                                       int64_t d_stride_t, float* dstate, void* workspace, size_t workspace_bytes,
                                       spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, B, L, D, &eb)) return rc;
  if (B == 0 || D == 0) return SPK_OK;
  SPK_REQUIRE(L == 0 || (x != nullptr && gate != nullptr && dx != nullptr && dgate != nullptr),
              "x, gate, dx and dgate must be non-null");
  SPK_REQUIRE(L <= spk::kRecChunk || carry != nullptr, "the forward pass's carry is needed above %d steps",
              spk::kRecChunk);
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(gh, eb) &&
                  spk::aligned_to(dx, eb) && spk::aligned_to(dgate, eb) && spk::aligned_to(state, 4) &&
                  spk::aligned_to(lengths, 4) && spk::aligned_to(carry, 4) && spk::aligned_to(glast, 4) &&
                  spk::aligned_to(dstate, 4),
              "tensors must be aligned to their elements");
  if (int rc = spk::rec_workspace_check(B, L, D, workspace, workspace_bytes)) return rc;
  spk::RecArgs a{};
  a.x = x;
  a.gate = gate;
  a.gh = gh;
  a.h0 = state;
  a.glast = glast;
  a.lengths = lengths;
  a.carry = const_cast<float*>(carry);
  a.dx = dx;
  a.dgate = dgate;
  a.dh0 = dstate;
  a.B = B;
  a.L = L;
  a.D = D;
  a.x_b = x_stride_b;
  a.x_t = x_stride_t;
  a.g_b = g_stride_b;
  a.g_t = g_stride_t;
  a.h_b = gh_stride_b;
  a.h_t = gh_stride_t;
  a.o_b = d_stride_b;
  a.o_t = d_stride_t;
  const bool aligned = D % 4 == 0 && spk::rec_aligned(x, eb, x_stride_b, x_stride_t) &&
                       spk::rec_aligned(gate, eb, g_stride_b, g_stride_t) &&
                       spk::rec_aligned(gh, eb, gh_stride_b, gh_stride_t) &&
                       spk::rec_aligned(dx, eb, d_stride_b, d_stride_t) &&
                       spk::rec_aligned(dgate, eb, d_stride_b, d_stride_t) && spk::aligned_to(state, 16) &&
                       spk::aligned_to(glast, 16) && spk::aligned_to(carry, 16) && spk::aligned_to(dstate, 16);
  cudaStream_t st = (cudaStream_t)stream;
  spk::RecPlan p{};
  spk::rec_plan(&a, &p,
                x_stride_b == D && g_stride_b == D && d_stride_b == D && (gh == nullptr || gh_stride_b == D),
                workspace);
  SPK_REC_LAUNCH(recurrence_backward_kernel);
  return SPK_OK;
}

extern "C" int spk_recurrence_step(const void* x, const void* gate, int dtype, int form, int64_t n,
                                   const float* state, void* out, float* new_state, spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, n, 1, 1, &eb)) return rc;
  if (n == 0) return SPK_OK;
  SPK_REQUIRE(x != nullptr && gate != nullptr && state != nullptr && out != nullptr && new_state != nullptr,
              "x, gate, state, out and new_state must be non-null");
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(out, eb) &&
                  spk::aligned_to(state, 4) && spk::aligned_to(new_state, 4),
              "tensors must be aligned to their elements");
  const unsigned blocks = (unsigned)spk::ceil_div(n, 256);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    spk::with_form(form, [&](auto f) {
      spk::recurrence_step_kernel<E, decltype(f)><<<blocks, 256, 0, (cudaStream_t)stream>>>(
          static_cast<const E*>(x), static_cast<const E*>(gate), state, n, static_cast<E*>(out), new_state);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
  return SPK_OK;
}
