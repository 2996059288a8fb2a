// Rotary positions: the first R of a head's D dimensions, taken as R/2 points of the plane, are turned by angles that grow
// with the token's position:
//     t_i = position * frequency_i
//     y_a = (x_a cos t_i - x_b sin t_i) g,   y_b = (x_b cos t_i + x_a sin t_i) g,   (a, b) = (i, i + R/2) or (2i, 2i + 1)
// and the other D - R dimensions are copied.  The gradient is the same map with -t_i (a rotation's transpose), so one kernel
// serves both directions; q and k (which may have fewer heads) go through one launch.
//
// Bound: memory, 2 x (heads of q and k) x D elements per token; the angles cost R/2 sincos per TOKEN, shared by all its heads.
// A warp takes one token: its lanes form the token's angles together (through shared memory), each lane keeps the few that
// belong to its 16 bytes of a row (16 + 16 for pairs half a row apart) in registers and walks over the heads with them, four
// rows' accesses in flight, the first of them issued before the angles.  With few tokens a token's heads are split over
// several warps.  There is no table of angles in memory: none has to be built, kept or bounded, and any position works.
// Measured, bf16, 16384 tokens x (32 + 8) heads x 128, 336 MB: a block per few tokens with the angles read from shared
// memory for every row 102 us (bank conflicts, 37 % occupancy); this form 56 us = 6.0 TB/s, 0.92 of a plain copy's rate, with
// 80 registers a thread (six blocks of an SM; the compiler's own choice of 128 would leave four).
// The angle is formed and reduced in 64 bits: at position 10^6 an fp32 product is off by 0.06 radians.  What is left, at most
// pi, is evaluated in fp32 with the first-order term of what its rounding drops: cosine and sine are right to about 2^-24.
#include <algorithm>

#include "kernels.cuh"

namespace elsa {

namespace {

constexpr int kRotaryWarps = 4, kRotaryThreads = 32 * kRotaryWarps;
constexpr int kInFlight = 4;
constexpr int kAnglesMax = 256;                      // angles of 32 lanes: at most 8 each

struct RotaryParams {
  const void* x[2]; void* y[2];                      // q and k; x[1] null: only q
  Strides xs[2], ys[2];
  int heads[2];
  const double* frequencies;
  const void* positions; int position_bytes; int64_t psb, psn;     // position_bytes 0: a row's index is its position
  int64_t tokens;                                    // batch * n
  int n, head_dim, rotary_dim, in_place;
  float magnitude, sign;
  int splits, split_heads;                           // warps of one token and heads of each
};

// W elements as they are in memory: 16 bytes as one access (in four registers until they are used), or one by one
template <typename T, int W, int V> struct RotaryVec { T e[W]; };
template <typename T, int W> struct RotaryVec<T, W, 16 / static_cast<int>(sizeof(T))> { uint4 e; };

__device__ __forceinline__ float2 cos_sin(double angle) {
  constexpr double two_pi_hi = 6.283185307179586, two_pi_lo = 2.4492935982947064e-16;
  const double turns = rint(angle * 0.15915494309189535);
  const double r = fma(-turns, two_pi_lo, fma(-turns, two_pi_hi, angle));
  // (in half turns: sincospif needs no reduction of its own, whose path for large arguments would cost local memory)
  const double h = r * 0.3183098861837907;
  const float hi = static_cast<float>(h), lo = static_cast<float>((h - static_cast<double>(hi)) * 3.141592653589793);
  float s, c;
  sincospif(hi, &s, &c);
  return make_float2(fmaf(-lo, s, c), fmaf(lo, c, s));
}

// V: elements of one access (16 bytes, or one element where rows, strides or R do not allow that).  A row of D elements is
// `rot_items` turned items (half layout: V elements at i and V at i + R/2; neighbours: V at i, at least a pair) and then
// copied ones, V elements each; rows of more than 32 items are walked 32 items at a time.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, 6)
rotary_kernel(const RotaryParams prm) {
  constexpr int W = INTERLEAVED && V == 1 ? 2 : V;   // elements of an item's access
  constexpr int A = INTERLEAVED ? W / 2 : W;         // angles of an item
  using Vec = RotaryVec<T, W, V>;
  using Copy = RotaryVec<T, V, V>;
  auto elements = [](const Vec& v) { return reinterpret_cast<const T*>(&v); };
  __shared__ float2 shared_angles[kRotaryWarps][kAnglesMax];
  const int lane = threadIdx.x & 31;
  float2* angles = shared_angles[threadIdx.x >> 5];
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRotaryWarps + (threadIdx.x >> 5);
  const int64_t t = unit / prm.splits;
  if (t >= prm.tokens) return;                       // (no barrier of the block follows)
  const int64_t b = t / prm.n, r = t - b * prm.n;
  const int h0 = static_cast<int>(unit - t * prm.splits) * prm.split_heads;
  const int h1 = min(prm.heads[0] + prm.heads[1], h0 + prm.split_heads);
  const T* src0 = static_cast<const T*>(prm.x[0]) + b * prm.xs[0].b + r * prm.xs[0].r;
  const T* src1 = static_cast<const T*>(prm.x[1]) + b * prm.xs[1].b + r * prm.xs[1].r;
  T* dst0 = static_cast<T*>(prm.y[0]) + b * prm.ys[0].b + r * prm.ys[0].r;
  T* dst1 = static_cast<T*>(prm.y[1]) + b * prm.ys[1].b + r * prm.ys[1].r;
  auto source = [&](int head) { return head < prm.heads[0] ? src0 + head * prm.xs[0].h : src1 + (head - prm.heads[0]) * prm.xs[1].h; };
  auto target = [&](int head) { return head < prm.heads[0] ? dst0 + head * prm.ys[0].h : dst1 + (head - prm.heads[0]) * prm.ys[1].h; };

  const int half = prm.rotary_dim / 2;
  const int rot_items = half / A;
  const int row_items = rot_items + (prm.in_place ? 0 : (prm.head_dim - prm.rotary_dim) / V);
  for (int first = 0; first < row_items; first += 32) {
    const int width = min(32, row_items - first), rows = 32 / width;
    const int item = first + lane % width, sub = lane / width;
    const bool turned = item < rot_items;
    const int e0 = turned ? item * W : prm.rotary_dim + (item - rot_items) * V;
    const int end = sub < rows ? h1 : 0;             // (lanes beyond the last whole row of a pass do nothing)
    Vec x[kInFlight], y[kInFlight];
    auto load = [&](int head0) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int head = head0 + u * rows;
        if (head >= end) continue;
        const T* p = source(head) + e0;
        if (turned) {
          x[u] = *reinterpret_cast<const Vec*>(p);
          if (!INTERLEAVED) y[u] = *reinterpret_cast<const Vec*>(p + half);
        } else {
          *reinterpret_cast<Copy*>(&x[u]) = *reinterpret_cast<const Copy*>(p);
        }
      }
    };
    load(h0 + sub);
    // the angles of this chunk's turned items, A consecutive ones each
    int64_t pos = r;
    if (prm.position_bytes == 8) pos = static_cast<const int64_t*>(prm.positions)[b * prm.psb + r * prm.psn];
    else if (prm.position_bytes == 4) pos = static_cast<const int32_t*>(prm.positions)[b * prm.psb + r * prm.psn];
    const int n_angles = max(0, min(width, rot_items - first)) * A;
    __syncwarp();
    for (int i = lane; i < n_angles; i += 32) {
      const float2 v = cos_sin(static_cast<double>(pos) * prm.frequencies[first * A + i]);
      angles[i] = make_float2(v.x * prm.magnitude, v.y * prm.magnitude * prm.sign);
    }
    __syncwarp();
    float2 cs[A];
#pragma unroll
    for (int e = 0; e < A; ++e) cs[e] = turned ? angles[(item - first) * A + e] : make_float2(1.f, 0.f);

    for (int head0 = h0 + sub; head0 < end; ) {
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        const int head = head0 + u * rows;
        if (head >= end) continue;
        T* p = target(head) + e0;
        if (!turned) {
          *reinterpret_cast<Copy*>(p) = *reinterpret_cast<const Copy*>(&x[u]);
          continue;
        }
        Vec o0, o1;
#pragma unroll
        for (int e = 0; e < A; ++e) {
          const float x0 = to_f32<T>(elements(x[u])[INTERLEAVED ? 2 * e : e]);
          const float x1 = to_f32<T>(INTERLEAVED ? elements(x[u])[2 * e + 1] : elements(y[u])[e]);
          const T a = from_f32<T>(x0 * cs[e].x - x1 * cs[e].y), c = from_f32<T>(x1 * cs[e].x + x0 * cs[e].y);
          reinterpret_cast<T*>(&o0)[INTERLEAVED ? 2 * e : e] = a;
          if (INTERLEAVED) reinterpret_cast<T*>(&o0)[2 * e + 1] = c;
          else reinterpret_cast<T*>(&o1)[e] = c;
        }
        *reinterpret_cast<Vec*>(p) = o0;
        if (!INTERLEAVED) *reinterpret_cast<Vec*>(p + half) = o1;
      }
      head0 += kInFlight * rows;
      load(head0);
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
  // with fewer tokens than eight warps for each SM a token's heads are split, down to one row of each lane
  const int all_heads = prm.heads[0] + prm.heads[1];
  const int v = wide ? kVec : 1;
  const int row_items = prm.rotary_dim / (interleaved ? std::max(2, v) : 2 * v) + (prm.in_place ? 0 : (prm.head_dim - prm.rotary_dim) / v);
  const int rows = 32 / std::min(32, row_items);
  const int64_t wanted = std::max<int64_t>(1, 8ll * sm_count() / prm.tokens);
  prm.split_heads = static_cast<int>(std::max<int64_t>(rows, cdiv64(all_heads, wanted)));
  prm.splits = static_cast<int>(cdiv64(all_heads, prm.split_heads));
  const int64_t blocks = cdiv64(prm.tokens * prm.splits, kRotaryWarps);
  if (blocks > 0x7fffffffll) return ELSA_ERR_UNSUPPORTED;
  const auto kernel = wide ? (interleaved ? &rotary_kernel<T, kVec, true> : &rotary_kernel<T, kVec, false>)
                           : (interleaved ? &rotary_kernel<T, 1, true> : &rotary_kernel<T, 1, false>);
  kernel<<<static_cast<unsigned>(blocks), kRotaryThreads, 0, st>>>(prm);
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
