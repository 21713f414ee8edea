// Device helpers shared by the serving kernels.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"
#include "serve.h"

namespace tttj {

// mbar_wait with the timer read only every 64 polls: reading it between polls costs more than
// the hand-over that is waited for.  Bounded like mbar_wait (limit_ns, or *abort).
__device__ __forceinline__ bool srv_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint64_t limit_ns) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (abort != nullptr && *abort) return false;
    if (globaltimer_ns() - t0 > limit_ns) return false;
  }
}

// A wait gave up: the call's status word, and the word that the device's next call looks at.
__device__ __forceinline__ void srv_report_timeout(int* status, int* timeout_host) {
  report_status(status, SRV_DEV_TIMEOUT);
  *reinterpret_cast<volatile int*>(timeout_host) = SRV_DEV_TIMEOUT;
}

template <bool BF16>
__device__ __forceinline__ uint32_t srv_pack(float a, float b) {
  if constexpr (BF16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    return pack_half2(a, b);
  }
}

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, uint32_t bar, int c0, int c1,
                                            int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// 32 bytes, 32-byte aligned.
__device__ __forceinline__ void srv_st_v8(void* to, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Whether one of the two 16-bit floats of a word is infinite or NaN.
template <bool BF16>
__device__ __forceinline__ bool srv_nonfinite(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}
// z + w * 0 for two 16-bit floats.
template <bool BF16>
__device__ __forceinline__ uint32_t srv_fma_zero(uint32_t w, uint32_t z) {
  uint32_t d;
  if constexpr (BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(z));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(w), "r"(0u), "r"(z));
  return d;
}
template <bool BF16>
__device__ __forceinline__ float srv_to_float(uint32_t half_bits) {
  if constexpr (BF16) return __uint_as_float(half_bits << 16);
  return __half2float(__ushort_as_half((unsigned short)half_bits));
}

// max(a, b, c), NaN if any of them is.
__device__ __forceinline__ float srv_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipe, as exp2_fma2 but as exact as ex2.approx (degree 5: max relative
// error 2.1e-7 in fp32 Horner arithmetic, coefficients fitted for this library by a Remez exchange
// on the relative error) and for every x: infinity where 2^x is none, 0 below 2^-125.5, NaN for
// NaN (2^j multiplies, since adding it into the bits of a NaN would give a number).  The
// polynomial is twice 2^f and the scale 2^(j-1), a normal number for j = rint(x) up to 128 and 0
// for j = -126, to which x is clamped from below.
__device__ __forceinline__ float2 exp2_fine2(float2 x) {
  float a, b;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(x.x), "f"(-126.0f));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(x.y), "f"(-126.0f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(128.0f));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(b) : "f"(b), "f"(128.0f));
  const unsigned long long xm = pk2(a, b);
  const unsigned long long magic = pk2(12582912.0f, 12582912.0f);
  const unsigned long long t = add2p(xm, magic);  // rint(x) in the low mantissa bits
  const unsigned long long f = sub2p(xm, sub2p(t, magic));
  unsigned long long p = fma2p(f, pk2(2.655294490e-03f, 2.655294490e-03f), pk2(1.9351081922e-02f, 1.9351081922e-02f));
  p = fma2p(f, p, pk2(1.1101426184e-01f, 1.1101426184e-01f));
  p = fma2p(f, p, pk2(4.804424048e-01f, 4.804424048e-01f));
  p = fma2p(f, p, pk2(1.386293888e+00f, 1.386293888e+00f));
  p = fma2p(f, p, pk2(2.000000238e+00f, 2.000000238e+00f));
  const float2 tf = upk2(t);
  return upk2(mul2p(p, pk2(__int_as_float((__float_as_int(tf.x) << 23) + 0x3f000000),
                           __int_as_float((__float_as_int(tf.y) << 23) + 0x3f000000))));
}

// tmem_wait_ld for a load whose registers are first used after other work: naming them keeps
// the compiler from moving a use in front of the wait.
__device__ __forceinline__ void tmem_wait_ld_of(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld_of(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
      :
      : "memory");
}

// Natural log-sum-exp of a row from its maximum (log2 domain) and sum: -inf for a row that
// sees no key, NaN where its scores hold one.
__device__ __forceinline__ float srv_lse(float top, float sum) {
  if (top == -INFINITY) return sum == 0.f ? -INFINITY : sum;
  return (top + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace tttj
