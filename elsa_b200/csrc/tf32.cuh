// fp32 products on the tensor cores' tf32 instruction (mma.sync m16n8k8, which reads the upper 19 bits of its operands): every operand x
// is taken as hi + lo, hi = x cut to tf32's 11 significant bits and lo = x - hi (exact), rounded to as many, and a b = hi hi + hi lo +
// lo hi.  lo is below 2^-10 of x, so an operand is right to 2^-21 of its size and what is left out, lo lo, is below 2^-20 of the
// product and 2^-22 of it on average; sums are fp32.  (Both parts rounded would be better by a third and take 5 % longer, for dQ
// at (1, 4 heads, 1000 tokens, 64 / 128, causal); cvt.rna, which runs at a fraction of the ALU's rate, 16 %.)  Three
// instructions of 1024 multiply-adds take the place of 32 FMAs of each thread and a quarter of their shared-memory reads.
#pragma once

#include "common.cuh"

namespace elsa {
namespace tf32 {

struct Split { uint32_t hi, lo; };

__device__ __forceinline__ Split split(float x) {
  Split s;
  s.hi = __float_as_uint(x) & 0xffffe000u;
  s.lo = __float_as_uint(x - __uint_as_float(s.hi)) + 0x1000u;      // (half a step of tf32: the instruction's cut rounds)
  return s;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d[16 x 8] += a[16 x 8] b[8 x 8].  The instruction cuts its sums instead of rounding them, always towards zero: three of them in a row are
// added to the running sum by an FADD, which rounds (a chain of them over 1000 keys lost 2 bits: 3.9e-6 against 8e-7 for dK).
__device__ __forceinline__ void mma3(float (&d)[4], const Split (&a)[4], const Split (&b)[2]) {
  float t[4] = {0.f, 0.f, 0.f, 0.f};
  mma(t, a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[0].hi, b[1].hi);
  mma(t, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].lo, b[1].lo);
  mma(t, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].hi, b[1].hi);
#pragma unroll
  for (int e = 0; e < 4; ++e) d[e] += t[e];
}

// Fragments of a warp's lane (r = lane / 4, q = lane % 4).  Matrices stand in shared memory row by row; a pitch of 4 mod 32 floats
// keeps every access below free of bank conflicts.
// A, rows r and r + 8, columns q and q + 4 of the 16 x 8 block at `p`
__device__ __forceinline__ void load_a(Split (&a)[4], const float* p, int pitch, int lane) {
  const float* s = p + (lane >> 2) * pitch + (lane & 3);
  a[0] = split(s[0]); a[1] = split(s[8 * pitch]); a[2] = split(s[4]); a[3] = split(s[8 * pitch + 4]);
}
// B of a product with the transpose: b[k][n] = p[n][k]
__device__ __forceinline__ void load_bt(Split (&b)[2], const float* p, int pitch, int lane) {
  const float* s = p + (lane >> 2) * pitch + (lane & 3);
  b[0] = split(s[0]); b[1] = split(s[4]);
}
// An accumulator block [16 x 8] as the A operand of the next product, and the rows of B that go with it: a lane's accumulator
// columns are 2q and 2q + 1 where the A operand has q and q + 4, so the eight products of a sum are taken in that order
__device__ __forceinline__ void acc_as_a(Split (&a)[4], const float (&d)[4]) {
  a[0] = split(d[0]); a[1] = split(d[2]); a[2] = split(d[1]); a[3] = split(d[3]);
}
__device__ __forceinline__ void load_b(Split (&b)[2], const float* p, int pitch, int lane) {
  const float* s = p + 2 * (lane & 3) * pitch + (lane >> 2);
  b[0] = split(s[0]); b[1] = split(s[pitch]);
}

// ROWS rows of a matrix of any type into shared memory as fp32 by THREADS threads, eight for each row, four columns at a time; rows from n
// on and columns from dim to COLS are zeros.  fetch and put apart: the loads can be on their way while the tile before is used.
template <typename T, int THREADS, int ROWS, int COLS>
struct Rows {
  static constexpr int kPass = THREADS / 8, kPasses = (ROWS + kPass - 1) / kPass, kSteps = COLS / 32, kRegs = kPasses * kSteps * 4;
  const T* base; int64_t stride; int n, dim;
  bool vec;                                             // (uniform) four elements in one access

  __device__ __forceinline__ Rows(const void* p, int64_t offset, int64_t stride_, int n_, int dim_)
      : base(static_cast<const T*>(p) + offset), stride(stride_), n(n_), dim(dim_) {
    vec = dim % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(base) & (4 * sizeof(T) - 1)) == 0;
  }
  __device__ __forceinline__ void fetch(float (&v)[kRegs], int x0) const {
    const int c = static_cast<int>(threadIdx.x) % 8 * 4;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = static_cast<int>(threadIdx.x) / 8 + i * kPass, r = x0 + row;
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        const int col = c + 32 * e;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (row < ROWS && r < n && col < dim) {
          const T* src = base + r * stride + col;
          if (vec) {
            Vec4<T>::load(src, x);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col + j < dim) x[j] = to_f32<T>(src[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) v[(i * kSteps + e) * 4 + j] = x[j];
      }
    }
  }
  static __device__ __forceinline__ void put(float* dst, int pitch, const float (&v)[kRegs]) {
    const int c = static_cast<int>(threadIdx.x) % 8 * 4;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = static_cast<int>(threadIdx.x) / 8 + i * kPass;
      if (row >= ROWS) continue;
#pragma unroll
      for (int e = 0; e < kSteps; ++e)
        *reinterpret_cast<float4*>(dst + row * pitch + c + 32 * e) =
            make_float4(v[(i * kSteps + e) * 4], v[(i * kSteps + e) * 4 + 1], v[(i * kSteps + e) * 4 + 2], v[(i * kSteps + e) * 4 + 3]);
    }
  }
  __device__ __forceinline__ void load(float* dst, int pitch, int x0) const {
    float v[kRegs];
    fetch(v, x0);
    put(dst, pitch, v);
  }
};

}  // namespace tf32
}  // namespace elsa
