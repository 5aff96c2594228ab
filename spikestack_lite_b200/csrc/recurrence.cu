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

constexpr int kRecChunk = 64;  // steps between the states kept for the backward pass

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

// The decay of a step as one float per form: `coeff` from the gate, `step` the
// new state, `back` the gradient that passes the step, dx and dgate the
// gradients of its inputs.
struct GateForm {
  __device__ static float coeff(float gate) { return gate; }
  __device__ static float step(float h, float a, float x) { return fmaf(a, h, x); }
  __device__ static float back(float g, float a) { return a * g; }
  __device__ static float dx(float g, float) { return g; }
  __device__ static float dgate(float g, float, float h, float) { return g * h; }
};

// Leaky form: whichever of a and q = 1 - a is at most one half, its sign bit
// set when it is a.  Both ends of the gate keep their relative accuracy: a
// slow channel's q and a fast channel's a are never differences from 1.
struct LeakyForm {
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
  __device__ static float back(float g, float c) { return is_a(c) ? -c * g : fmaf(-c, g, g); }
  __device__ static float dx(float g, float c) { return is_a(c) ? fmaf(c, g, g) : c * g; }
  __device__ static float dgate(float g, float c, float h, float x) {
    const float s = fabsf(c);
    return g * (h - x) * fmaf(-s, s, s);
  }
};

__device__ __forceinline__ int64_t rec_len(const RecArgs& a, int64_t b) {
  if (a.lengths == nullptr) return a.L;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : (n > a.L ? a.L : n);
}

template <typename E, typename Form>
__global__ void __launch_bounds__(128) recurrence_kernel(RecArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.B * a.D) return;
  const int64_t b = i / a.D, d = i - b * a.D, len = rec_len(a, b);
  const E* x = static_cast<const E*>(a.x) + b * a.x_b + d;
  const E* g = static_cast<const E*>(a.gate) + b * a.g_b + d;
  E* out = static_cast<E*>(a.h) + b * a.h_b + d;
  float h = a.h0 != nullptr ? a.h0[i] : 0.0f;
  for (int64_t t = 0; t < a.L; ++t) {
    if (t > 0 && t % kRecChunk == 0 && a.carry != nullptr) a.carry[(t / kRecChunk - 1) * a.B * a.D + i] = h;
    if (t < len) h = Form::step(h, Form::coeff(elem_to_f32(g[t * a.g_t])), elem_to_f32(x[t * a.x_t]));
    out[t * a.h_t] = elem_from_f32<E>(t < len ? h : 0.0f);
  }
  a.last[i] = h;
}

template <typename E, typename Form>
__global__ void __launch_bounds__(128) recurrence_backward_kernel(RecArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= a.B * a.D) return;
  const int64_t b = i / a.D, d = i - b * a.D, len = rec_len(a, b);
  const E* x = static_cast<const E*>(a.x) + b * a.x_b + d;
  const E* gate = static_cast<const E*>(a.gate) + b * a.g_b + d;
  const E* gh = a.gh != nullptr ? static_cast<const E*>(a.gh) + b * a.h_b + d : nullptr;
  E* dx = static_cast<E*>(a.dx) + b * a.o_b + d;
  E* dg = static_cast<E*>(a.dgate) + b * a.o_b + d;
  for (int64_t t = len; t < a.L; ++t) {
    dx[t * a.o_t] = elem_from_f32<E>(0.0f);
    dg[t * a.o_t] = elem_from_f32<E>(0.0f);
  }
  float c = a.glast != nullptr ? a.glast[i] : 0.0f;  // gradient reaching h_t from later steps
  float hb[kRecChunk];
  for (int64_t k = ceil_div(len, kRecChunk) - 1; k >= 0; --k) {
    const int64_t t0 = k * kRecChunk, n = min64(len - t0, kRecChunk);
    float h = k > 0 ? a.carry[(k - 1) * a.B * a.D + i] : (a.h0 != nullptr ? a.h0[i] : 0.0f);
    for (int64_t j = 0; j < n; ++j) {
      hb[j] = h;
      h = Form::step(h, Form::coeff(elem_to_f32(gate[(t0 + j) * a.g_t])), elem_to_f32(x[(t0 + j) * a.x_t]));
    }
    for (int64_t j = n - 1; j >= 0; --j) {
      const int64_t t = t0 + j;
      const float q = Form::coeff(elem_to_f32(gate[t * a.g_t])), xv = elem_to_f32(x[t * a.x_t]);
      const float g = c + (gh != nullptr ? elem_to_f32(gh[t * a.h_t]) : 0.0f);
      dx[t * a.o_t] = elem_from_f32<E>(Form::dx(g, q));
      dg[t * a.o_t] = elem_from_f32<E>(Form::dgate(g, q, hb[j], xv));
      c = Form::back(g, q);
    }
  }
  if (a.dh0 != nullptr) a.dh0[i] = c;
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
  return SPK_OK;
}

}  // namespace spk

extern "C" int spk_recurrence_chunk(void) { return spk::kRecChunk; }

extern "C" size_t spk_recurrence_workspace_bytes(int64_t B, int64_t L, int64_t D) {
  (void)B;
  (void)L;
  (void)D;
  return 0;
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
  (void)workspace;
  (void)workspace_bytes;
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
  const unsigned blocks = (unsigned)spk::ceil_div(B * D, 128);
  spk::with_elem(dtype, [&](auto e) {
    spk::with_form(form, [&](auto f) {
      spk::recurrence_kernel<decltype(e), decltype(f)><<<blocks, 128, 0, (cudaStream_t)stream>>>(a);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
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
  (void)workspace;
  (void)workspace_bytes;
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
  const unsigned blocks = (unsigned)spk::ceil_div(B * D, 128);
  spk::with_elem(dtype, [&](auto e) {
    spk::with_form(form, [&](auto f) {
      spk::recurrence_backward_kernel<decltype(e), decltype(f)><<<blocks, 128, 0, (cudaStream_t)stream>>>(a);
    });
  });
  SPK_LAUNCH_CHECK();
  spk::count_launch(1);
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
