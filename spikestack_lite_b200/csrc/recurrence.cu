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
//
// Bound: HBM (x and gate read, h written; backward x, gate and gh read, dx and
// dgate written: h is run again from the states kept every 64 or 128 steps) for
// short recurrences and fp32; the latency of one tile's passes and joins for
// long 16-bit ones, where an SM holds 16 warps of some 25 instructions per
// element.  Measured, leaky, against the time the bytes need:
//   4 planes of 65536x512 fp32          284 us, all of it
//   64x2048x512  bf16  89 us forward (69 %), 163 us backward (63 %)
//   4x32768x512  bf16 141 us forward (44 %), 239 us backward (43 %)
//   4x32768x512  fp32 199 us forward (62 %), 354 us backward (58 %)
//   64x2048x512  fp32 149 us forward (83 %), 289 us backward (71 %)
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
  float* carry;           // [chunks - 1, B, D]: the states between tiles along time; or null
  void* dx;
  void* dgate;
  float* dh0;
  int64_t B, L, D;
  int64_t x_b, x_t, g_b, g_t, h_b, h_t, o_b, o_t;  // strides in elements (h: h or gh; o: dx and dgate)
};

struct RecPlan {
  int64_t chains, groups;  // chains = B * groups of neighbouring channels
  int64_t tiles, chunks;   // blocks' tiles (short), tiles along time (long)
  int wt, cols;            // warps along time (short); channels per chain
  int steps, cluster;      // steps per warp, blocks per chain (long)
};

// Two neighbouring channels: sm_100 multiplies and adds fp32 numbers in pairs.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 two(float f) { return F2{f, f}; }
__device__ __forceinline__ uint64_t f2_bits(F2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ F2 f2_of(uint64_t r) {
  F2 a;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a.x), "=f"(a.y) : "l"(r));
  return a;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return f2_of(r);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return f2_of(r);
}
__device__ __forceinline__ F2 sub2(F2 a, F2 b) { return fma2(b, two(-1.0f), a); }

// The decay of one or more steps as one float per form: `coeff` from the gate,
// `step` the new state, `apply` A h + H for a joined decay A, `join` the decay
// of two in a row, `back` the gradient that passes a step, `grads` that and
// the gradients of the step's inputs (from `base` of the state before and x).
// A warp's steps are joined by `open`, one `more` per step and `close`.
// kept_gate is the gate, kept the decay, of a step that keeps the state.
struct GateForm {
  __device__ static float kept_gate() { return 1.0f; }
  __device__ static float kept() { return 1.0f; }
  __device__ static float open() { return 1.0f; }
  __device__ static float coeff(float gate) { return gate; }
  __device__ static F2 coeff(F2 gate, F2*) { return gate; }
  __device__ static F2 more(F2 acc, F2 a, F2) { return mul2(acc, a); }
  __device__ static float close(float acc) { return acc; }
  __device__ static float apply(float a, float h, float H) { return fmaf(a, h, H); }
  __device__ static float join(float a, float b) { return a * b; }
  __device__ static float step(float h, float a, float x) { return fmaf(a, h, x); }
  __device__ static F2 step(F2 h, F2 a, F2 x) { return fma2(a, h, x); }
  __device__ static F2 back(F2 g, F2 a) { return mul2(a, g); }
  __device__ static F2 base(F2 h, F2) { return h; }
  __device__ static F2 grads(F2 g, F2 a, F2 base, F2* dx, F2* dgate) {
    *dx = g;
    *dgate = mul2(g, base);
    return mul2(a, g);
  }
};

// Leaky form, fp32 tensors.  A decay, of one step or of several, is whichever
// of A and Q = 1 - A is at most one half, the sign bit set when it is A:
// neither a slow channel's Q nor a fast channel's A is a difference from 1.
// Over a warp's steps, with e = exp(-gate) and a = 1 / (1 + e), the product of
// decays is 1 / (1 + E) with E = prod (1 + e) - 1, a sum of positive terms
// (kept finite: below 2^-124 a joined decay is as good as 0).
struct LeakyForm {
  __device__ static float kept_gate() { return __int_as_float(0x7f800000); }  // q = 0
  __device__ static float kept() { return 0.0f; }
  __device__ static float open() { return 0.0f; }
  __device__ static bool is_a(float c) { return __float_as_int(c) < 0; }
  // the decay of a step; *e (when wanted) becomes exp(-gate)
  __device__ static float coeff(float gate, float* e = nullptr) {
    const float small = expf(-fabsf(gate));
    if (e != nullptr) *e = gate < 0.0f ? rcp_fast(fmaxf(small, 0x1p-124f)) : small;
    return copysignf(small * rcp_fast(1.0f + small), gate);
  }
  __device__ static F2 coeff(F2 gate, F2* e) {
    return e != nullptr ? F2{coeff(gate.x, &e->x), coeff(gate.y, &e->y)} : F2{coeff(gate.x), coeff(gate.y)};
  }
  __device__ static F2 more(F2 acc, F2, F2 e) {
    const F2 r = fma2(acc, e, add2(acc, e));
    return F2{fminf(r.x, 0x1p124f), fminf(r.y, 0x1p124f)};
  }
  __device__ static float close(float acc) {
    const float a = rcp_fast(1.0f + acc);
    return acc <= 1.0f ? acc * a : -a;
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
  __device__ static float step(float h, float c, float x) {
    const bool fast = is_a(c);  // x + a (h - x), else h + q (x - h)
    const float base = fast ? x : h;
    return fmaf(fabsf(c), (fast ? h : x) - base, base);
  }
  __device__ static F2 step(F2 h, F2 c, F2 x) { return F2{step(h.x, c.x, x.x), step(h.y, c.y, x.y)}; }
  __device__ static float back(float g, float c) { return is_a(c) ? -c * g : fmaf(-c, g, g); }
  __device__ static F2 back(F2 g, F2 c) { return F2{back(g.x, c.x), back(g.y, c.y)}; }
  __device__ static float dx(float g, float c) { return is_a(c) ? fmaf(c, g, g) : c * g; }
  __device__ static F2 base(F2 h, F2 x) { return sub2(h, x); }
  __device__ static F2 grads(F2 g, F2 c, F2 base, F2* dx_, F2* dgate) {
    const F2 s = F2{fabsf(c.x), fabsf(c.y)};
    *dx_ = F2{dx(g.x, c.x), dx(g.y, c.y)};
    *dgate = mul2(mul2(g, base), sub2(s, mul2(s, s)));
    return back(g, c);
  }
};

// Leaky form, 16-bit tensors: a decay is Q = 1 - A, and exp the hardware's.  A
// slow channel is as exact as above; a fast one's result is off by a rounding
// of the state before it, and the weights are off by some 2^-21, far below the
// 2^-9 or 2^-12 that the tensors carry.  It takes half the instructions, and
// the 16-bit kernels are bound by those, the fp32 ones by memory.
struct LeakyHalfForm {
  __device__ static float kept_gate() { return __int_as_float(0x7f800000); }
  __device__ static float kept() { return 0.0f; }
  __device__ static float open() { return 0.0f; }
  __device__ static float coeff(float gate) { return rcp_fast(1.0f + ex2_fast(gate * 1.4426950409f)); }
  __device__ static F2 coeff(F2 gate, F2*) {
    const F2 t = mul2(gate, two(1.4426950409f)), d = add2(F2{ex2_fast(t.x), ex2_fast(t.y)}, two(1.0f));
    return F2{rcp_fast(d.x), rcp_fast(d.y)};
  }
  __device__ static F2 more(F2 acc, F2 c, F2) { return step(acc, c, two(1.0f)); }
  __device__ static float close(float acc) { return acc; }
  __device__ static float apply(float c, float h, float H) { return fmaf(-c, h, h) + H; }
  __device__ static float join(float c, float d) { return fmaf(-c, d, c) + d; }
  __device__ static float step(float h, float c, float x) { return fmaf(c, x - h, h); }
  __device__ static F2 step(F2 h, F2 c, F2 x) { return fma2(c, sub2(x, h), h); }
  __device__ static F2 back(F2 g, F2 c) { return sub2(g, mul2(c, g)); }
  __device__ static F2 base(F2 h, F2 x) { return sub2(h, x); }
  __device__ static F2 grads(F2 g, F2 c, F2 base, F2* dx, F2* dgate) {
    *dx = mul2(c, g);
    *dgate = mul2(*dx, mul2(base, sub2(two(1.0f), c)));
    return sub2(g, *dx);
  }
};

__device__ __forceinline__ int64_t rec_len(const RecArgs& a, int64_t b) {
  if (a.lengths == nullptr) return a.L;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : (n > a.L ? a.L : n);
}

// ---- tiles
// A warp holds S steps of 32 V neighbouring channels of one batch row (a
// "chain" along time) in registers, V channels per lane, and a block is 8
// warps.  Each warp reduces its steps to one affine map h -> A h + H, the maps
// meet in shared memory, and every warp then runs its steps once more from its
// own start, in the order of the definition: states are exact in the sense of
// the sequential recurrence within a warp's steps, and joined by A h + H
// between.  Blocks go from tile to tile: while one is worked on, the next
// one's inputs are on their way to shared memory (each lane copies what it
// will read itself, so that needs no barrier), 2 blocks per SM.
constexpr int kRecWarps = 8;
constexpr int kRecThreads = 32 * kRecWarps;
constexpr int kRecMaxCluster = 16;

// The lane's V channels of `n` (at most 32 V) starting at p: neighbours moved
// as one access (ALIGNED), or every 32nd.
template <int V>
struct Cols {
  float v[V];
  __device__ __forceinline__ F2 pair(int i) const { return F2{v[2 * i], v[2 * i + 1]}; }
  __device__ __forceinline__ void pair(int i, F2 p) {
    v[2 * i] = p.x;
    v[2 * i + 1] = p.y;
  }
};

template <int V, bool ALIGNED>
__device__ __forceinline__ int rec_col(int lane, int i) {
  return ALIGNED ? V * lane + i : lane + 32 * i;
}

template <int V, bool ALIGNED, typename E>
__device__ __forceinline__ Cols<V> rec_load(const E* p, int lane, int n, float other) {
  Cols<V> q;
  if (ALIGNED) {
    if (V * lane < n) {
      const Pack<E, V> e = load_pack<E, V>(p + V * lane);
#pragma unroll
      for (int i = 0; i < V; ++i) q.v[i] = elem_to_f32(e.e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) q.v[i] = other;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) q.v[i] = lane + 32 * i < n ? elem_to_f32(p[lane + 32 * i]) : other;
  }
  return q;
}

template <int V, bool ALIGNED, typename E>
__device__ __forceinline__ void rec_store(E* p, int lane, int n, const Cols<V>& q) {
  if (ALIGNED) {
    if (V * lane < n) store_pack<E, V>(p + V * lane, pack_f32<E, V>(q.v));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane + 32 * i < n) p[lane + 32 * i] = elem_from_f32<E>(q.v[i]);
  }
}

// Maps in shared memory are in the lanes' order: channel i of a lane at V lane + i.
template <int V>
__device__ __forceinline__ Cols<V> cols_ld(const float* p, int lane) {
  const Pack<float, V> e = load_pack<float, V>(p + V * lane);
  Cols<V> q;
#pragma unroll
  for (int i = 0; i < V; ++i) q.v[i] = e.e[i];
  return q;
}
template <int V>
__device__ __forceinline__ void cols_st(float* p, int lane, const Cols<V>& q) {
  Pack<float, V> e;
#pragma unroll
  for (int i = 0; i < V; ++i) e.e[i] = q.v[i];
  store_pack<float, V>(p + V * lane, e);
}

// Where a warp's part of a tile lies: S steps from t0, of which the first
// `steps` are before the row's end and `room` before the tensor's, n channels
// from col (all counts 0: nothing there, the state stays).
struct RecSpot {
  int64_t b, col, t0;
  int n, steps, room;
};

// `len`: the valid steps of row q->b; the spot's n channels and t0 are set.
template <int S>
__device__ __forceinline__ void rec_extent(int64_t len, int64_t L, RecSpot* q) {
  q->steps = (int)max64(min64(len - q->t0, S), 0);
  q->room = (int)max64(min64(L - q->t0, S), 0);
}

// An input may be fetched ahead where a lane's piece is what cp.async moves.
template <typename E, int V, bool ALIGNED>
__host__ __device__ constexpr bool rec_ahead() {
  return ALIGNED && V * sizeof(E) >= 4;
}

// The S pieces of one input on their way; a step behind the row's end gets `other`.
template <typename E, int V, int S>
__device__ __forceinline__ void rec_copy(E* stage, const void* base, int64_t stride_b, int64_t stride_t,
                                         const RecSpot& q, int lane, float other) {
  const E* p = static_cast<const E*>(base) + q.b * stride_b + q.t0 * stride_t + q.col + V * lane;
  const int steps = V * lane < q.n ? q.steps : 0;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    if (j < steps) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(stage + j * 32 * V)), "l"(p),
                   "n"(V * sizeof(E) >= 4 ? V * sizeof(E) : 4)
                   : "memory");
    } else {
      Pack<E, V> e;
#pragma unroll
      for (int i = 0; i < V; ++i) e.e[i] = elem_from_f32<E>(other);
      store_pack<E, V>(stage + j * 32 * V, e);
    }
    p += stride_t;
  }
}

template <typename E, int V, int S, bool ALIGNED>
__device__ __forceinline__ void rec_take(Cols<V>* v, const E* stage, const void* base, int64_t stride_b,
                                         int64_t stride_t, const RecSpot& q, int lane, float other) {
  if (rec_ahead<E, V, ALIGNED>()) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const Pack<E, V> e = load_pack<E, V>(stage + j * 32 * V);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j].v[i] = elem_to_f32(e.e[i]);
    }
  } else {
    const E* p = static_cast<const E*>(base) + q.b * stride_b + q.t0 * stride_t + q.col;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      v[j] = rec_load<V, ALIGNED>(p, lane, j < q.steps ? q.n : 0, other);
      p += stride_t;
    }
  }
}

template <typename E, int V, int S, bool ALIGNED>
__host__ __device__ constexpr size_t rec_stage_bytes(int tensors) {
  return rec_ahead<E, V, ALIGNED>() ? (size_t)tensors * kRecWarps * S * 32 * V * sizeof(E) : 0;
}

// A lane's inputs of a forward tile and the places they travel through.
template <typename E, int V, int S, bool ALIGNED>
struct RecInputs {
  E* stage;
  int lane;
  static constexpr int kStep = kRecWarps * S * 32 * V;  // between the tensors' stages

  __device__ __forceinline__ RecInputs(unsigned char* smem, int warp, int lane_)
      : stage(reinterpret_cast<E*>(smem) + warp * S * 32 * V + V * lane_), lane(lane_) {}
  __device__ __forceinline__ void ask(const RecArgs& a, const RecSpot& q, float kept_gate, bool backward) const {
    if constexpr (rec_ahead<E, V, ALIGNED>()) {
      rec_copy<E, V, S>(stage, a.gate, a.g_b, a.g_t, q, lane, kept_gate);
      rec_copy<E, V, S>(stage + kStep, a.x, a.x_b, a.x_t, q, lane, 0.0f);
      if (backward && a.gh != nullptr) rec_copy<E, V, S>(stage + 2 * kStep, a.gh, a.h_b, a.h_t, q, lane, 0.0f);
    }
  }
  __device__ __forceinline__ void wait() const {
    if constexpr (rec_ahead<E, V, ALIGNED>()) asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __device__ __forceinline__ void gate(const RecArgs& a, const RecSpot& q, Cols<V>* v, float other) const {
    rec_take<E, V, S, ALIGNED>(v, stage, a.gate, a.g_b, a.g_t, q, lane, other);
  }
  __device__ __forceinline__ void x(const RecArgs& a, const RecSpot& q, Cols<V>* v) const {
    rec_take<E, V, S, ALIGNED>(v, stage + kStep, a.x, a.x_b, a.x_t, q, lane, 0.0f);
  }
  __device__ __forceinline__ void gh(const RecArgs& a, const RecSpot& q, Cols<V>* v) const {
    if (a.gh != nullptr) {
      rec_take<E, V, S, ALIGNED>(v, stage + 2 * kStep, a.gh, a.h_b, a.h_t, q, lane, 0.0f);
    } else {
#pragma unroll
      for (int j = 0; j < S; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) v[j].v[i] = 0.0f;
    }
  }
};

template <int V>
__device__ __forceinline__ Cols<V> cols_of(float f) {
  Cols<V> q;
#pragma unroll
  for (int i = 0; i < V; ++i) q.v[i] = f;
  return q;
}

template <typename Form, int V>
__device__ __forceinline__ void cols_apply(const float* A, const float* H, int lane, Cols<V>* h) {
  const Cols<V> pA = cols_ld<V>(A, lane), pH = cols_ld<V>(H, lane);
#pragma unroll
  for (int i = 0; i < V; ++i) h->v[i] = Form::apply(pA.v[i], h->v[i], pH.v[i]);
}

// The gates become decays, and the warp's steps one map (A, H).
template <typename Form, int V, int S>
__device__ __forceinline__ void rec_reduce(Cols<V>* c, const Cols<V>* u, Cols<V>* A, Cols<V>* H) {
  *A = cols_of<V>(Form::open());
  *H = cols_of<V>(0.0f);
#pragma unroll
  for (int j = 0; j < S; ++j)
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      F2 e;
      const F2 d = Form::coeff(c[j].pair(i), &e);
      c[j].pair(i, d);
      H->pair(i, Form::step(H->pair(i), d, u[j].pair(i)));
      A->pair(i, Form::more(A->pair(i), d, e));
    }
#pragma unroll
  for (int i = 0; i < V; ++i) A->v[i] = Form::close(A->v[i]);
}

template <typename Form, int V, int S>
__device__ __forceinline__ void rec_coeffs(Cols<V>* c) {
#pragma unroll
  for (int j = 0; j < S; ++j)
#pragma unroll
    for (int i = 0; i < V / 2; ++i) c[j].pair(i, Form::coeff(c[j].pair(i), nullptr));
}

// The gradient's map of the warp's steps (its decay is A too).
template <typename Form, int V, int S>
__device__ __forceinline__ Cols<V> rec_reduce_back(const Cols<V>* c, const Cols<V>* g) {
  Cols<V> G = cols_of<V>(0.0f);
#pragma unroll
  for (int j = S - 1; j >= 0; --j)
#pragma unroll
    for (int i = 0; i < V / 2; ++i) G.pair(i, Form::back(add2(g[j].pair(i), G.pair(i)), c[j].pair(i)));
  return G;
}

// The warp's states from h on, written; h becomes the state behind them.
template <typename E, typename Form, int V, int S, bool ALIGNED>
__device__ __forceinline__ void rec_run_forward(const RecArgs& a, const RecSpot& q, const Cols<V>* c, const Cols<V>* u,
                                                Cols<V>* h, int lane) {
  E* out = static_cast<E*>(a.h) + q.b * a.h_b + q.t0 * a.h_t + q.col;
#pragma unroll
  for (int j = 0; j < S; ++j) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) h->pair(i, Form::step(h->pair(i), c[j].pair(i), u[j].pair(i)));
    if (j < q.steps)
      rec_store<V, ALIGNED>(out, lane, q.n, *h);
    else if (j < q.room)
      rec_store<V, ALIGNED>(out, lane, q.n, cols_of<V>(0.0f));
    out += a.h_t;
  }
}

// The warp's states from h on; what dgate needs of them takes x's place.
template <typename Form, int V, int S>
__device__ __forceinline__ void rec_replay(const Cols<V>* c, Cols<V>* u, Cols<V> h) {
#pragma unroll
  for (int j = 0; j < S; ++j)
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const F2 before = h.pair(i);
      h.pair(i, Form::step(before, c[j].pair(i), u[j].pair(i)));
      u[j].pair(i, Form::base(before, u[j].pair(i)));
    }
}

// The warp's gradients from the one that reaches its last step, written;
// `later` becomes the one that reaches the step before its first.
template <typename E, typename Form, int V, int S, bool ALIGNED>
__device__ __forceinline__ void rec_run_back(const RecArgs& a, const RecSpot& q, const Cols<V>* c, const Cols<V>* u,
                                             const Cols<V>* g, Cols<V>* later, int lane) {
  const int64_t end = q.b * a.o_b + (q.t0 + S - 1) * a.o_t + q.col;
  E *dx = static_cast<E*>(a.dx) + end, *dg = static_cast<E*>(a.dgate) + end;
#pragma unroll
  for (int j = S - 1; j >= 0; --j) {
    Cols<V> ox, og;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      F2 px, pg;
      later->pair(i, Form::grads(add2(g[j].pair(i), later->pair(i)), c[j].pair(i), u[j].pair(i), &px, &pg));
      ox.pair(i, px);
      og.pair(i, pg);
    }
    if (j < q.steps) {
      rec_store<V, ALIGNED>(dx, lane, q.n, ox);
      rec_store<V, ALIGNED>(dg, lane, q.n, og);
    } else if (j < q.room) {
      rec_store<V, ALIGNED>(dx, lane, q.n, cols_of<V>(0.0f));
      rec_store<V, ALIGNED>(dg, lane, q.n, cols_of<V>(0.0f));
    }
    dx -= a.o_t;
    dg -= a.o_t;
  }
}

// ---- up to 64 steps: `wt` warps of a block along time (the fewest powers of
// two that hold them), 8 / wt along chains; blocks take every gridDim-th tile.
template <int S>
__device__ __forceinline__ RecSpot rec_short_spot(const RecArgs& a, const RecPlan& p, int64_t tile, int warp) {
  RecSpot q{};
  const int64_t chain = tile * (kRecWarps / p.wt) + warp / p.wt;
  if (chain >= p.chains) return q;
  q.b = chain / p.groups;
  q.col = (chain - q.b * p.groups) * 128;
  q.n = (int)min64(a.D - q.col, 128);
  q.t0 = (warp % p.wt) * S;
  rec_extent<S>(rec_len(a, q.b), a.L, &q);
  return q;
}

template <typename E, typename Form, int S, bool ALIGNED>
__global__ void __launch_bounds__(kRecThreads, 2) recurrence_short_kernel(RecArgs a, RecPlan p) {
  constexpr int V = 4;
  extern __shared__ __align__(16) unsigned char rec_smem[];
  __shared__ __align__(16) float mA[2][kRecWarps][32 * V], mH[2][kRecWarps][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % p.wt;
  const RecInputs<E, V, S, ALIGNED> in(rec_smem, warp, lane);
  RecSpot q = rec_short_spot<S>(a, p, blockIdx.x, warp);
  in.ask(a, q, Form::kept_gate(), false);
  int round = 0;
  for (int64_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x, round ^= 1) {
    Cols<V> c[S], u[S];
    in.wait();
    in.gate(a, q, c, Form::kept_gate());
    in.x(a, q, u);
    const RecSpot next = rec_short_spot<S>(a, p, tile + gridDim.x, warp);
    in.ask(a, next, Form::kept_gate(), false);
    Cols<V> h = cols_of<V>(0.0f);
    if (a.h0 != nullptr) h = rec_load<V, ALIGNED>(a.h0 + q.b * a.D + q.col, lane, q.n, 0.0f);
    if (p.wt > 1) {
      Cols<V> A, H;
      rec_reduce<Form, V, S>(c, u, &A, &H);
      cols_st<V>(mA[round][warp], lane, A);
      cols_st<V>(mH[round][warp], lane, H);
      __syncthreads();
      for (int k = warp - w; k < warp; ++k) cols_apply<Form, V>(mA[round][k], mH[round][k], lane, &h);
    } else {
      rec_coeffs<Form, V, S>(c);
    }
    rec_run_forward<E, Form, V, S, ALIGNED>(a, q, c, u, &h, lane);
    if (w + 1 == p.wt) rec_store<V, ALIGNED>(a.last + q.b * a.D + q.col, lane, q.n, h);
    q = next;
  }
}

template <typename E, typename Form, int S, bool ALIGNED>
__global__ void __launch_bounds__(kRecThreads, 2) recurrence_short_backward_kernel(RecArgs a, RecPlan p) {
  constexpr int V = 4;
  extern __shared__ __align__(16) unsigned char rec_smem[];
  __shared__ __align__(16) float mA[kRecWarps][32 * V], mH[kRecWarps][32 * V], mG[kRecWarps][32 * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % p.wt;
  const RecInputs<E, V, S, ALIGNED> in(rec_smem, warp, lane);
  RecSpot q = rec_short_spot<S>(a, p, blockIdx.x, warp);
  in.ask(a, q, Form::kept_gate(), true);
  for (int64_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
    Cols<V> c[S], u[S], g[S];
    in.wait();
    in.gate(a, q, c, Form::kept_gate());
    in.x(a, q, u);
    in.gh(a, q, g);
    const RecSpot next = rec_short_spot<S>(a, p, tile + gridDim.x, warp);
    in.ask(a, next, Form::kept_gate(), true);
    Cols<V> h = cols_of<V>(0.0f), later = cols_of<V>(0.0f);
    if (a.h0 != nullptr) h = rec_load<V, ALIGNED>(a.h0 + q.b * a.D + q.col, lane, q.n, 0.0f);
    if (a.glast != nullptr) later = rec_load<V, ALIGNED>(a.glast + q.b * a.D + q.col, lane, q.n, 0.0f);
    if (p.wt > 1) {
      Cols<V> A, H;
      rec_reduce<Form, V, S>(c, u, &A, &H);
      cols_st<V>(mA[warp], lane, A);
      cols_st<V>(mH[warp], lane, H);
      cols_st<V>(mG[warp], lane, rec_reduce_back<Form, V, S>(c, g));
      __syncthreads();
      for (int k = warp - w; k < warp; ++k) cols_apply<Form, V>(mA[k], mH[k], lane, &h);
      for (int k = warp - w + p.wt - 1; k > warp; --k) cols_apply<Form, V>(mA[k], mG[k], lane, &later);
      __syncthreads();  // the maps are read: the next tile's may come
    } else {
      rec_coeffs<Form, V, S>(c);
    }
    rec_replay<Form, V, S>(c, u, h);
    rec_run_back<E, Form, V, S, ALIGNED>(a, q, c, u, g, &later, lane);
    if (a.dh0 != nullptr && w == 0) rec_store<V, ALIGNED>(a.dh0 + q.b * a.D + q.col, lane, q.n, later);
    q = next;
  }
}

// ---- longer sequences: one cluster of K blocks per chain walks along time,
// K tiles of 8 S steps at once.  Every block sends its tile's map to all of
// them (stores to the cluster's shared memory that count bytes on the
// receiver's barrier) and applies all K in time order, so each knows the state
// in front of its own tile and the one behind them all, which it carries on:
// no block waits for another cluster, x and gate are read once however few
// chains there are, and the order of every sum is fixed.
struct RecMeeting {
  float2* maps;  // [2][K][32 V] (A, H) by parity of the round and rank, behind the stages
  uint64_t* bar; // [2]
  int* abort;
};

constexpr size_t rec_meeting_bytes(int V, int K) { return K > 1 ? (size_t)2 * K * 32 * V * sizeof(float2) : 0; }

// Sends a block's map (of the warps' maps, in time order or in reverse), this
// thread's channel c, to every block's maps[parity][rank].
template <typename Form, int V>
__device__ __forceinline__ void rec_send(const RecMeeting& m, const float (*mA)[32 * V], const float (*mH)[32 * V],
                                         bool reverse, int parity, int rank, int K, int c) {
  float A = Form::kept(), H = 0.0f;
#pragma unroll
  for (int k = 0; k < kRecWarps; ++k) {
    const int w = reverse ? kRecWarps - 1 - k : k;
    H = Form::apply(mA[w][c], H, mH[w][c]);
    A = Form::join(A, mA[w][c]);
  }
  const uint32_t at = smem_u32(m.maps + (parity * K + rank) * 32 * V + c), bar = smem_u32(m.bar + parity);
  if (c == 0) mbar_arrive_expect_tx(m.bar + parity, (uint32_t)(K * 32 * V * sizeof(float2)));
  for (int k = 0; k < K; ++k) {
    uint32_t there, there_bar;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(k));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there_bar) : "r"(bar), "r"(k));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(there),
                 "f"(A), "f"(H), "r"(there_bar)
                 : "memory");
  }
}

// Applies the K maps of a round (in the order of ranks, or in reverse) to
// `state`, the one in front of them all; returns the one in front of this
// block's tile and moves `state` behind them.  A sender overwrites a map two
// rounds later, after it has received this block's map of the round between,
// which this thread sends when it is done here.
template <typename Form, int V>
__device__ __forceinline__ float rec_meet(const RecMeeting& m, bool reverse, int round, int rank, int K, int c,
                                          float* state) {
  mbar_wait<true>(m.bar + (round & 1), (round >> 1) & 1, m.abort, SPK_DEV_PIPE_TIMEOUT);
  const float2* maps = m.maps + (round & 1) * K * 32 * V + c;
  float s = *state, front = s;
#pragma unroll 4
  for (int k = 0; k < K; ++k) {
    const int r = reverse ? K - 1 - k : k;
    const float2 v = maps[r * 32 * V];
    if (r == rank) front = s;
    s = Form::apply(v.x, s, v.y);
  }
  *state = s;
  return front;
}

__device__ __forceinline__ void rec_meeting_open(const RecMeeting& m, int K) {
  if (K == 1) return;
  if (threadIdx.x == 0) {
    mbar_init(m.bar, 1);
    mbar_init(m.bar + 1, 1);
    *m.abort = 0;
    fence_barrier_init();
  }
  cluster_sync_all();
}

// The chain of a cluster, and a warp's spot in the tile `chunk` of it.
template <int V, int S>
struct RecChain {
  int64_t len, L;
  RecSpot q;
  int n;

  __device__ __forceinline__ RecChain(const RecArgs& a, const RecPlan& p, int64_t chain) : L(a.L) {
    q.b = chain / p.groups;
    q.col = (chain - q.b * p.groups) * (32 * V);
    n = (int)min64(a.D - q.col, 32 * V);
    len = rec_len(a, q.b);
  }
  __device__ __forceinline__ RecSpot at(int64_t chunk, int warp) const {
    RecSpot r = q;
    r.t0 = (chunk * kRecWarps + warp) * S;
    r.n = n;
    if (chunk >= 0)
      rec_extent<S>(len, L, &r);
    else
      r.steps = r.room = 0;  // in front of the first tile; behind the last, no step is left either
    return r;
  }
};

template <typename E, typename Form, int V, int S, bool ALIGNED>
__global__ void __launch_bounds__(kRecThreads, 2) recurrence_long_kernel(RecArgs a, RecPlan p) {
  extern __shared__ __align__(16) unsigned char rec_smem[];
  __shared__ __align__(16) float mA[2][kRecWarps][32 * V], mH[2][kRecWarps][32 * V], sC[32 * V];
  __shared__ uint64_t bars[2];
  __shared__ int abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = threadIdx.x;
  const int rank = (int)cluster_ctarank(), K = p.cluster;
  const int64_t chain = blockIdx.x / K;
  const RecMeeting meeting{reinterpret_cast<float2*>(rec_smem + rec_stage_bytes<E, V, S, ALIGNED>(2)), bars, &abort};
  rec_meeting_open(meeting, K);
  const RecInputs<E, V, S, ALIGNED> in(rec_smem, warp, lane);
  const RecChain<V, S> walk(a, p, chain);
  RecSpot q = walk.at(rank, warp);
  in.ask(a, q, Form::kept_gate(), false);
  const int width = walk.n, ch = rec_col<V, ALIGNED>(slot / V, slot % V);
  const bool joins = slot < 32 * V;  // this thread joins the tiles for channel ch
  float state = joins && ch < width && a.h0 != nullptr ? a.h0[q.b * a.D + q.col + ch] : 0.0f;
  int round = 0;
  for (int64_t first = 0; first < p.chunks; first += K, ++round) {
    const int64_t chunk = first + rank;
    Cols<V> c[S], u[S], A, H;
    in.wait();
    in.gate(a, q, c, Form::kept_gate());
    in.x(a, q, u);
    const RecSpot next = walk.at(chunk + K, warp);
    in.ask(a, next, Form::kept_gate(), false);
    rec_reduce<Form, V, S>(c, u, &A, &H);
    cols_st<V>(mA[round & 1][warp], lane, A);
    cols_st<V>(mH[round & 1][warp], lane, H);
    __syncthreads();
    if (joins) {
      float front = state;
      if (K > 1) {
        rec_send<Form, V>(meeting, mA[round & 1], mH[round & 1], false, round & 1, rank, K, slot);
        front = rec_meet<Form, V>(meeting, false, round, rank, K, slot, &state);
      } else {
#pragma unroll
        for (int k = 0; k < kRecWarps; ++k) state = Form::apply(mA[round & 1][k][slot], state, mH[round & 1][k][slot]);
      }
      sC[slot] = front;
      if (a.carry != nullptr && chunk > 0 && chunk < p.chunks && ch < width)
        a.carry[((chunk - 1) * a.B + q.b) * a.D + q.col + ch] = front;
    }
    __syncthreads();
    Cols<V> h = cols_ld<V>(sC, lane);
    for (int k = 0; k < warp; ++k) cols_apply<Form, V>(mA[round & 1][k], mH[round & 1][k], lane, &h);
    rec_run_forward<E, Form, V, S, ALIGNED>(a, q, c, u, &h, lane);
    q = next;
  }
  if (joins && rank == 0 && ch < width) a.last[q.b * a.D + q.col + ch] = state;
  if (K > 1) cluster_sync_all();  // maps may still be on their way here
}

// Backward: the same tiles from the end.  A tile runs its steps forward from
// the state the forward pass kept (h is not read back from memory, where it
// was rounded), and backwards from the gradient that reaches it, whose affine
// map has the same decay.
template <typename E, typename Form, int V, int S, bool ALIGNED>
__global__ void __launch_bounds__(kRecThreads, 2) recurrence_long_backward_kernel(RecArgs a, RecPlan p) {
  extern __shared__ __align__(16) unsigned char rec_smem[];
  __shared__ __align__(16) float mA[kRecWarps][32 * V], mH[kRecWarps][32 * V], mG[kRecWarps][32 * V];
  __shared__ __align__(16) float sC[32 * V];
  __shared__ uint64_t bars[2];
  __shared__ int abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = threadIdx.x;
  const int rank = (int)cluster_ctarank(), K = p.cluster;
  const int64_t chain = blockIdx.x / K;
  const RecMeeting meeting{reinterpret_cast<float2*>(rec_smem + rec_stage_bytes<E, V, S, ALIGNED>(3)), bars, &abort};
  rec_meeting_open(meeting, K);
  const RecInputs<E, V, S, ALIGNED> in(rec_smem, warp, lane);
  const int64_t top = (p.chunks - 1) / K * K;
  const RecChain<V, S> walk(a, p, chain);
  RecSpot q = walk.at(top + rank, warp);
  in.ask(a, q, Form::kept_gate(), true);
  const int width = walk.n, ch = rec_col<V, ALIGNED>(slot / V, slot % V);
  const bool joins = slot < 32 * V;
  float state = joins && ch < width && a.glast != nullptr ? a.glast[q.b * a.D + q.col + ch] : 0.0f;
  int round = 0;
  for (int64_t first = top; first >= 0; first -= K, ++round) {
    const int64_t chunk = first + rank;
    Cols<V> c[S], u[S], g[S], h;
    in.wait();
    in.gate(a, q, c, Form::kept_gate());
    in.x(a, q, u);
    in.gh(a, q, g);
    const RecSpot next = walk.at(chunk - K, warp);
    in.ask(a, next, Form::kept_gate(), true);
    {
      Cols<V> A, H;
      rec_reduce<Form, V, S>(c, u, &A, &H);
      cols_st<V>(mA[warp], lane, A);
      cols_st<V>(mH[warp], lane, H);
      cols_st<V>(mG[warp], lane, rec_reduce_back<Form, V, S>(c, g));
    }
    h = cols_of<V>(0.0f);
    const float* start = chunk > 0 ? a.carry + ((chunk - 1) * a.B + q.b) * a.D : a.h0 + q.b * a.D;
    if (chunk < p.chunks && (chunk > 0 || a.h0 != nullptr)) h = rec_load<V, ALIGNED>(start + q.col, lane, q.n, 0.0f);
    __syncthreads();
    if (K > 1 && joins) rec_send<Form, V>(meeting, mA, mG, true, round & 1, rank, K, slot);
    for (int k = 0; k < warp; ++k) cols_apply<Form, V>(mA[k], mH[k], lane, &h);
    rec_replay<Form, V, S>(c, u, h);
    if (joins) {
      float front = state;
      if (K > 1) {
        front = rec_meet<Form, V>(meeting, true, round, rank, K, slot, &state);
      } else {
#pragma unroll
        for (int k = kRecWarps - 1; k >= 0; --k) state = Form::apply(mA[k][slot], state, mG[k][slot]);
      }
      sC[slot] = front;
    }
    __syncthreads();
    Cols<V> later = cols_ld<V>(sC, lane);
    for (int k = kRecWarps - 1; k > warp; --k) cols_apply<Form, V>(mA[k], mG[k], lane, &later);
    __syncthreads();  // the maps are read: the next tile's may come
    rec_run_back<E, Form, V, S, ALIGNED>(a, q, c, u, g, &later, lane);
    q = next;
  }
  if (joins && rank == 0 && ch < width && a.dh0 != nullptr) a.dh0[q.b * a.D + q.col + ch] = state;
  if (K > 1) cluster_sync_all();  // maps may still be on their way here
}

// One step of the recurrence over rows of D cells: out (element type) and the
// new state (fp32; may be the old state's own buffer).
template <typename E, typename Form>
__global__ void __launch_bounds__(256) recurrence_step_kernel(const E* __restrict__ x, int64_t x_stride,
                                                              const E* __restrict__ gate, int64_t g_stride,
                                                              const float* state, int64_t n, int D,
                                                              E* __restrict__ out, float* new_state) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int64_t r = i / D, d = i - r * D;
  const float h =
      Form::step(state[i], Form::coeff(elem_to_f32(gate[r * g_stride + d])), elem_to_f32(x[r * x_stride + d]));
  out[i] = elem_from_f32<E>(h);
  new_state[i] = h;
}

template <typename E, typename F>
inline void with_form(int form, F&& f) {
  if (form == SPK_REC_GATE)
    f(GateForm{});
  else if constexpr (sizeof(E) == 4)
    f(LeakyForm{});
  else
    f(LeakyHalfForm{});
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
  SPK_REQUIRE(B < (1ll << 31) / (kRecMaxCluster * max64(ceil_div(D, 32), 1)),
              "too many rows (B=%lld, D=%lld)", (long long)B, (long long)D);
  return SPK_OK;
}

static bool rec_aligned(const void* p, size_t eb, int64_t stride_b, int64_t stride_t) {
  return aligned_to(p, 4 * eb) && stride_b % 4 == 0 && stride_t % 4 == 0;
}

// Shape of a long recurrence's tiles: 128 channels (V = 4 per lane) or 64 (V =
// 2), 8 or 16 steps per warp.  64 channels are twice the chains, 16 steps half
// the joins, and fp32's backward stages leave room for one block per SM beside
// 128-channel maps.  Forward and backward (which share the steps per tile), us:
//                          4 x 8        2 x 16       2 x 8
//   bf16  1x32768x512      86 / 132     70 / 127     84 / 128
//         4x32768x512     145 / 240    137 / 255    153 / 254
//         64x2048x512      90 / 165    119 / 241    127 / 224
//   fp32  4x32768x512     270 / 476    200 / 355    219 / 338
//         64x2048x512     147 / 383    172 / 324    174 / 289
struct RecShape {
  int cols, steps;
};

static RecShape rec_long_shape(int dtype, int64_t B, int64_t D, bool backward) {
  const int64_t chains = B * ceil_div(D, 128);
  if (dtype == SPK_F32) {
    if (chains < 64) return {64, 16};
    return backward ? RecShape{64, 8} : RecShape{128, 8};
  }
  return chains < 16 ? RecShape{64, 16} : RecShape{128, 8};
}

static int64_t rec_chunk(int dtype, int64_t B, int64_t L, int64_t D) {
  return L <= 64 ? 64 : kRecWarps * rec_long_shape(dtype, B, D, false).steps;
}

// Batch rows that follow one another like channels (no lengths, batch stride D
// everywhere) become channels first, so that narrow rows share a warp.
static RecPlan rec_plan(RecArgs* a, int dtype, bool backward, bool merge) {
  RecPlan p{};
  const int64_t chunk = rec_chunk(dtype, a->B, a->L, a->D);
  const RecShape shape = rec_long_shape(dtype, a->B, a->D, backward);
  p.cols = a->L <= 64 ? 128 : shape.cols;
  p.steps = shape.steps;
  if (merge && a->lengths == nullptr) {
    a->D *= a->B;
    a->B = 1;
  }
  p.groups = ceil_div(a->D, p.cols);
  p.chains = a->B * p.groups;
  p.chunks = max64(ceil_div(a->L, chunk), 1);
  p.wt = 1;
  while (p.wt < kRecWarps && (int64_t)p.wt * 8 < a->L) p.wt *= 2;
  p.tiles = ceil_div(p.chains, kRecWarps / p.wt);
  return p;
}

template <typename E, typename Form, int S, bool ALIGNED>
static cudaError_t rec_launch_short(bool backward, const RecArgs& a, const RecPlan& p, cudaStream_t st) {
  auto* const kernel =
      backward ? recurrence_short_backward_kernel<E, Form, S, ALIGNED> : recurrence_short_kernel<E, Form, S, ALIGNED>;
  const size_t smem = rec_stage_bytes<E, 4, S, ALIGNED>(backward ? 3 : 2);
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  kernel<<<(unsigned)min64(p.tiles, 2 * (int64_t)sm_count()), kRecThreads, smem, st>>>(a, p);
  return cudaGetLastError();
}

// Clusters of k blocks of a kernel that run at once, k = 1 .. 16 (0: none).
struct RecOccupancy {
  int clusters[kRecMaxCluster + 1];
};

template <typename K>
static cudaError_t rec_occupancy(K* kernel, int V, size_t stages, RecOccupancy* out) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)(stages + rec_meeting_bytes(V, kRecMaxCluster)));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  for (int k = 1; k <= kRecMaxCluster && e == cudaSuccess; ++k) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)k);
    cfg.blockDim = dim3(kRecThreads);
    cfg.dynamicSmemBytes = stages + rec_meeting_bytes(V, k);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)k;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    out->clusters[k] = 0;
    if (cudaOccupancyMaxActiveClusters(&out->clusters[k], kernel, &cfg) != cudaSuccess) {
      out->clusters[k] = 0;
      (void)cudaGetLastError();
    }
  }
  return e;
}

template <typename E, typename Form, int V, int S, bool ALIGNED, bool BACKWARD>
static cudaError_t rec_launch_long(const RecArgs& a, const RecPlan& p, cudaStream_t st) {
  auto* const kernel = [] {  // only the one that is launched is compiled
    if constexpr (BACKWARD)
      return &recurrence_long_backward_kernel<E, Form, V, S, ALIGNED>;
    else
      return &recurrence_long_kernel<E, Form, V, S, ALIGNED>;
  }();
  const size_t stages = rec_stage_bytes<E, V, S, ALIGNED>(BACKWARD ? 3 : 2);
  static PerDevice<RecOccupancy> cache;  // one per kernel
  RecOccupancy occ;
  cudaError_t e = cache.get(&occ, [&](RecOccupancy* o) { return rec_occupancy(kernel, V, stages, o); });
  if (e != cudaSuccess) return e;
  // The fewest blocks per chain that need the fewest rounds: every cluster
  // takes ceil(chunks / k) rounds, as many clusters at once as fit.
  RecPlan plan = p;
  plan.cluster = 1;
  int64_t best = 0;
  for (int k = 1; k <= kRecMaxCluster && k <= p.chunks; ++k) {
    if (occ.clusters[k] <= 0) continue;
    const int64_t rounds = ceil_div(p.chains, occ.clusters[k]) * ceil_div(p.chunks, k);
    if (best == 0 || rounds < best) {
      best = rounds;
      plan.cluster = k;
    }
  }
  return launch_dependent_cluster(kernel, dim3((unsigned)(p.chains * plan.cluster)), dim3(kRecThreads),
                                  stages + rec_meeting_bytes(V, plan.cluster), st, (unsigned)plan.cluster, false, a,
                                  plan);
}

template <typename E, typename Form, int V, int S, bool ALIGNED>
static cudaError_t rec_launch_long(bool backward, const RecArgs& a, const RecPlan& p, cudaStream_t st) {
  return backward ? rec_launch_long<E, Form, V, S, ALIGNED, true>(a, p, st)
                  : rec_launch_long<E, Form, V, S, ALIGNED, false>(a, p, st);
}

static int rec_run(bool backward, int dtype, int form, bool aligned, const RecArgs& a, const RecPlan& p,
                   cudaStream_t st) {
  cudaError_t rc = cudaSuccess;
  with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    with_form<E>(form, [&](auto f) {
      using F = decltype(f);
      if (a.L > 64 && p.cols == 64 && p.steps == 16) {
        rc = aligned ? rec_launch_long<E, F, 2, 16, true>(backward, a, p, st)
                     : rec_launch_long<E, F, 2, 16, false>(backward, a, p, st);
      } else if (a.L > 64) {
        if constexpr (sizeof(E) != 4)
          rc = aligned ? rec_launch_long<E, F, 4, 8, true>(backward, a, p, st)
                       : rec_launch_long<E, F, 4, 8, false>(backward, a, p, st);
        else if (backward)
          rc = aligned ? rec_launch_long<E, F, 2, 8, true, true>(a, p, st)
                       : rec_launch_long<E, F, 2, 8, false, true>(a, p, st);
        else
          rc = aligned ? rec_launch_long<E, F, 4, 8, true, false>(a, p, st)
                       : rec_launch_long<E, F, 4, 8, false, false>(a, p, st);
      }
      else if (a.L > 4)
        rc = aligned ? rec_launch_short<E, F, 8, true>(backward, a, p, st)
                     : rec_launch_short<E, F, 8, false>(backward, a, p, st);
      else
        rc = aligned ? rec_launch_short<E, F, 4, true>(backward, a, p, st)
                     : rec_launch_short<E, F, 4, false>(backward, a, p, st);
    });
  });
  if (rc != cudaSuccess) return fail(SPK_ECUDA, "recurrence launch failed: %s", cudaGetErrorString(rc));
  count_launch(1);
  return SPK_OK;
}

}  // namespace spk

extern "C" int64_t spk_recurrence_chunk(int dtype, int64_t B, int64_t L, int64_t D) {
  return B > 0 && L > 0 && D > 0 ? spk::rec_chunk(dtype, B, L, D) : 64;
}

extern "C" int spk_recurrence(const void* x, int64_t x_stride_b, int64_t x_stride_t, const void* gate,
                              int64_t g_stride_b, int64_t g_stride_t, int dtype, int form, int64_t B, int64_t L,
                              int64_t D, const float* state, const int32_t* lengths, void* h, int64_t h_stride_b,
                              int64_t h_stride_t, float* last, float* carry, spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, B, L, D, &eb)) return rc;
  if (B == 0 || D == 0) return SPK_OK;
  SPK_REQUIRE(last != nullptr && (L == 0 || (x != nullptr && gate != nullptr && h != nullptr)),
              "x, gate, h and last must be non-null");
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(h, eb) &&
                  spk::aligned_to(state, 4) && spk::aligned_to(lengths, 4) && spk::aligned_to(last, 4) &&
                  spk::aligned_to(carry, 4),
              "tensors must be aligned to their elements");
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
  const spk::RecPlan p = spk::rec_plan(&a, dtype, false, x_stride_b == D && g_stride_b == D && h_stride_b == D);
  return spk::rec_run(false, dtype, form, aligned, a, p, st);
}

extern "C" int spk_recurrence_backward(const void* x, int64_t x_stride_b, int64_t x_stride_t, const void* gate,
                                       int64_t g_stride_b, int64_t g_stride_t, const void* gh, int64_t gh_stride_b,
                                       int64_t gh_stride_t, int dtype, int form, int64_t B, int64_t L, int64_t D,
                                       const float* state, const int32_t* lengths, const float* carry,
                                       const float* glast, void* dx, void* dgate, int64_t d_stride_b,
                                       int64_t d_stride_t, float* dstate, spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, B, L, D, &eb)) return rc;
  if (B == 0 || D == 0) return SPK_OK;
  SPK_REQUIRE(L == 0 || (x != nullptr && gate != nullptr && dx != nullptr && dgate != nullptr),
              "x, gate, dx and dgate must be non-null");
  SPK_REQUIRE(L <= spk::rec_chunk(dtype, B, L, D) || carry != nullptr, "the forward pass's carry is needed above %lld steps",
              (long long)spk::rec_chunk(dtype, B, L, D));
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(gh, eb) &&
                  spk::aligned_to(dx, eb) && spk::aligned_to(dgate, eb) && spk::aligned_to(state, 4) &&
                  spk::aligned_to(lengths, 4) && spk::aligned_to(carry, 4) && spk::aligned_to(glast, 4) &&
                  spk::aligned_to(dstate, 4),
              "tensors must be aligned to their elements");
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
  const spk::RecPlan p = spk::rec_plan(
      &a, dtype, true, x_stride_b == D && g_stride_b == D && d_stride_b == D && (gh == nullptr || gh_stride_b == D));
  return spk::rec_run(true, dtype, form, aligned, a, p, st);
}

extern "C" int spk_recurrence_step(const void* x, int64_t x_stride, const void* gate, int64_t g_stride, int dtype,
                                   int form, int64_t rows, int64_t D, const float* state, void* out, float* new_state,
                                   spk_stream_t stream) {
  size_t eb = 0;
  if (int rc = spk::rec_check(dtype, form, rows, 1, D, &eb)) return rc;
  if (rows == 0 || D == 0) return SPK_OK;
  SPK_REQUIRE(x != nullptr && gate != nullptr && state != nullptr && out != nullptr && new_state != nullptr,
              "x, gate, state, out and new_state must be non-null");
  SPK_REQUIRE(spk::aligned_to(x, eb) && spk::aligned_to(gate, eb) && spk::aligned_to(out, eb) &&
                  spk::aligned_to(state, 4) && spk::aligned_to(new_state, 4),
              "tensors must be aligned to their elements");
  const unsigned blocks = (unsigned)spk::ceil_div(rows * D, 256);
  spk::with_elem(dtype, [&](auto e) {
    using E = decltype(e);
    spk::with_form<E>(form, [&](auto f) {
      spk::recurrence_step_kernel<E, decltype(f)><<<blocks, 256, 0, (cudaStream_t)stream>>>(
          static_cast<const E*>(x), x_stride, static_cast<const E*>(gate), g_stride, state, rows * D, (int)D,
          static_cast<E*>(out), new_state);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
  return SPK_OK;
}
