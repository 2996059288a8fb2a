// Rotary positions: the first R of a head's D dimensions, taken as R/2 points of the plane, are turned by angles that grow
// with the token's position:
//     t_i = position * frequency_i
//     y_a = (x_a cos t_i - x_b sin t_i) g,   y_b = (x_b cos t_i + x_a sin t_i) g,   (a, b) = (i, i + R/2) or (2i, 2i + 1)
// and the other D - R dimensions are copied.  The gradient is the same map with -t_i (a rotation's transpose), so one kernel
// serves both directions; q and k (which may have fewer heads) go through one launch.
//
// Bound: memory, 2 x (heads of q and k) x D elements per token; the angles cost R/2 sincos per TOKEN, shared by all its heads.
// Each block takes a few consecutive tokens, puts their cosines and sines into shared memory and then streams the rows of all
// heads through, 16 bytes per access, up to four accesses of each thread in flight.  There is no table of angles in memory:
// none has to be built, kept or bounded, and any position works.
// The angle is formed and reduced in 64 bits: at position 10^6 an fp32 product is off by 0.06 radians.  What is left, at most
// pi, is evaluated in fp32 with the first-order term of what its rounding drops: cosine and sine are right to about 2^-24.
#include <algorithm>

#include "kernels.cuh"

namespace elsa {

namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokensMax = 32;                 // tokens of one block (their angles: at most 32 x 64 x 8 bytes)
constexpr int kInFlight = 4;

struct RotaryParams {
  const void* x[2]; void* y[2];                      // q and k; x[1] null: only q
  Strides xs[2], ys[2];
  int heads[2];
  const double* frequencies;
  const void* positions; int position_bytes; int64_t psb, psn;     // position_bytes 0: a row's index is its position
  int64_t tokens;                                    // batch * n
  int n, head_dim, rotary_dim, in_place;
  float magnitude, sign;
  int tokens_per_block;
};

// W elements, A of them aligned as one access
template <typename T, int W, int A> struct alignas(sizeof(T) * A) RotaryVec { T e[W]; };

__device__ __forceinline__ float2 cos_sin(double angle) {
  constexpr double two_pi_hi = 6.283185307179586, two_pi_lo = 2.4492935982947064e-16;
  const double turns = rint(angle * 0.15915494309189535);
  const double r = fma(-turns, two_pi_lo, fma(-turns, two_pi_hi, angle));
  const float hi = static_cast<float>(r), lo = static_cast<float>(r - static_cast<double>(hi));
  float s, c;
  sincosf(hi, &s, &c);
  return make_float2(fmaf(-lo, s, c), fmaf(lo, c, s));
}

// V: elements of one access (16 bytes, or one element where rows, strides or R do not allow that).  A row of D elements is
// `rot_items` turned items (half layout: V elements at i and V at i + R/2; neighbours: V at i, at least a pair) and then
// `copy_items` copied ones.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const RotaryParams prm) {
  constexpr int W = INTERLEAVED && V == 1 ? 2 : V;   // elements of an item's access
  extern __shared__ float2 angles[];                 // [token][R/2]: cosine and sine, times the magnitude
  const int half = prm.rotary_dim / 2;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * prm.tokens_per_block;
  const int nt = static_cast<int>(min(static_cast<int64_t>(prm.tokens_per_block), prm.tokens - t0));
  for (int i = threadIdx.x; i < nt * half; i += kRotaryThreads) {
    const int tok = i / half, f = i - tok * half;
    const int64_t t = t0 + tok, b = t / prm.n, r = t - b * prm.n;
    int64_t pos = r;
    if (prm.position_bytes == 8) pos = static_cast<const int64_t*>(prm.positions)[b * prm.psb + r * prm.psn];
    else if (prm.position_bytes == 4) pos = static_cast<const int32_t*>(prm.positions)[b * prm.psb + r * prm.psn];
    const float2 cs = cos_sin(static_cast<double>(pos) * prm.frequencies[f]);
    angles[i] = make_float2(cs.x * prm.magnitude, cs.y * prm.magnitude * prm.sign);
  }
  __syncthreads();

  const int rot_items = INTERLEAVED ? prm.rotary_dim / W : half / V;
  const int copy_items = prm.in_place ? 0 : (prm.head_dim - prm.rotary_dim) / V;
  const int row_items = rot_items + copy_items;
  const int all_heads = prm.heads[0] + prm.heads[1];
  const int total = nt * all_heads * row_items;
  using Vec = RotaryVec<T, W, V>;
  using Copy = RotaryVec<T, V, V>;

  for (int base = threadIdx.x; base < total; base += kInFlight * kRotaryThreads) {
    Vec a[kInFlight], c[kInFlight];
    T* dst[kInFlight];
    int item_of[kInFlight], tok_of[kInFlight];
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int idx = base + u * kRotaryThreads;
      item_of[u] = -1;
      if (idx >= total) continue;
      const int row = idx / row_items, item = idx - row * row_items;
      const int tok = row / all_heads, head = row - tok * all_heads;
      const int which = head >= prm.heads[0];
      const int h = which ? head - prm.heads[0] : head;
      const int64_t t = t0 + tok, b = t / prm.n, r = t - b * prm.n;
      const Strides xs = prm.xs[which], ys = prm.ys[which];
      const T* src = static_cast<const T*>(prm.x[which]) + b * xs.b + h * xs.h + r * xs.r;
      dst[u] = static_cast<T*>(prm.y[which]) + b * ys.b + h * ys.h + r * ys.r;
      item_of[u] = item;
      tok_of[u] = tok;
      if (item >= rot_items) {
        const int e = prm.rotary_dim + (item - rot_items) * V;
        *reinterpret_cast<Copy*>(&a[u]) = *reinterpret_cast<const Copy*>(src + e);
      } else {
        a[u] = *reinterpret_cast<const Vec*>(src + item * W);
        if (!INTERLEAVED) c[u] = *reinterpret_cast<const Vec*>(src + half + item * W);
      }
    }
#pragma unroll
    for (int u = 0; u < kInFlight; ++u) {
      const int item = item_of[u];
      if (item < 0) continue;
      if (item >= rot_items) {
        const int e = prm.rotary_dim + (item - rot_items) * V;
        *reinterpret_cast<Copy*>(dst[u] + e) = *reinterpret_cast<const Copy*>(&a[u]);
        continue;
      }
      if (INTERLEAVED) {
        const float2* cs = angles + tok_of[u] * half + item * (W / 2);
        Vec o;
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
          const float x0 = to_f32<T>(a[u].e[2 * e]), x1 = to_f32<T>(a[u].e[2 * e + 1]);
          o.e[2 * e] = from_f32<T>(x0 * cs[e].x - x1 * cs[e].y);
          o.e[2 * e + 1] = from_f32<T>(x1 * cs[e].x + x0 * cs[e].y);
        }
        *reinterpret_cast<Vec*>(dst[u] + item * W) = o;
      } else {
        const float2* cs = angles + tok_of[u] * half + item * W;
        Vec o0, o1;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float x0 = to_f32<T>(a[u].e[e]), x1 = to_f32<T>(c[u].e[e]);
          o0.e[e] = from_f32<T>(x0 * cs[e].x - x1 * cs[e].y);
          o1.e[e] = from_f32<T>(x1 * cs[e].x + x0 * cs[e].y);
        }
        *reinterpret_cast<Vec*>(dst[u] + item * W) = o0;
        *reinterpret_cast<Vec*>(dst[u] + half + item * W) = o1;
      }
    }
  }
}

template <typename T>
int rotary_t(RotaryParams& prm, bool interleaved, cudaStream_t st) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  bool wide = prm.head_dim % kVec == 0 && (interleaved ? prm.rotary_dim : prm.rotary_dim / 2) % kVec == 0;
  for (int i = 0; i < (prm.x[1] ? 2 : 1); ++i) {
    const Strides &a = prm.xs[i], &b = prm.ys[i];
    wide = wide && ((a.b | a.h | a.r | b.b | b.h | b.r) % kVec) == 0 &&
           ((reinterpret_cast<uintptr_t>(prm.x[i]) | reinterpret_cast<uintptr_t>(prm.y[i])) & 15u) == 0;
  }
  const int v = wide ? kVec : 1;
  // tokens of a block: about four items for each thread, but at least two blocks for each SM while there are tokens for that
  const int items = ((interleaved ? prm.rotary_dim / (v == 1 ? 2 : v) : prm.rotary_dim / 2 / v) +
                     (prm.in_place ? 0 : (prm.head_dim - prm.rotary_dim) / v)) * (prm.heads[0] + prm.heads[1]);
  int64_t per = (kInFlight * kRotaryThreads + items - 1) / items;
  per = std::min<int64_t>(per, std::max<int64_t>(1, prm.tokens / (2 * sm_count())));
  prm.tokens_per_block = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(per, kRotaryTokensMax)));
  const int64_t blocks = cdiv64(prm.tokens, prm.tokens_per_block);
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  const size_t smem = static_cast<size_t>(prm.tokens_per_block) * (prm.rotary_dim / 2) * sizeof(float2);
  const auto kernel = wide ? (interleaved ? &rotary_kernel<T, kVec, true> : &rotary_kernel<T, kVec, false>)
                           : (interleaved ? &rotary_kernel<T, 1, true> : &rotary_kernel<T, 1, false>);
  kernel<<<static_cast<unsigned>(blocks), kRotaryThreads, smem, st>>>(prm);
  ELSA_LAUNCH_CHECK();
  return ELSA_OK;
}

}  // namespace

int rotary(const void* q, void* q_out, const int64_t* qs, int q_heads, const void* k, void* k_out, const int64_t* ks, int k_heads,
           const double* frequencies, const void* positions, int position_bytes, int64_t psb, int64_t psn, double magnitude,
           int dtype, int batch, int n, int head_dim, int rotary_dim, int interleaved, int inverse, cudaStream_t st) {
  RotaryParams prm{};
  prm.x[0] = q; prm.y[0] = q_out; prm.heads[0] = q_heads;
  prm.xs[0] = Strides{qs[0], qs[1], qs[2]}; prm.ys[0] = Strides{qs[3], qs[4], qs[5]};
  prm.in_place = q == q_out;
  if (k) {
    prm.x[1] = k; prm.y[1] = k_out; prm.heads[1] = k_heads;
    prm.xs[1] = Strides{ks[0], ks[1], ks[2]}; prm.ys[1] = Strides{ks[3], ks[4], ks[5]};
    prm.in_place = prm.in_place && k == k_out;
  }
  prm.frequencies = frequencies; prm.positions = positions; prm.position_bytes = position_bytes; prm.psb = psb; prm.psn = psn;
  prm.tokens = static_cast<int64_t>(batch) * n;
  prm.n = n; prm.head_dim = head_dim; prm.rotary_dim = rotary_dim;
  prm.magnitude = static_cast<float>(magnitude); prm.sign = inverse ? -1.f : 1.f;
  if (dtype == ELSA_F32) return rotary_t<float>(prm, interleaved != 0, st);
  if (dtype == ELSA_F16) return rotary_t<__half>(prm, interleaved != 0, st);
  return rotary_t<__nv_bfloat16>(prm, interleaved != 0, st);
}

}  // namespace elsa
