// Rows into and out of the paged 4-bit cache (layout and numbers: q4.cuh).
//
// Both directions stream: 2 bytes a channel on one side, 9/16 on the other, a
// maximum and a rounding between.  65,521 rows of 8 kv heads are 344 MB each way
// together with their source or result, 52.6 us of HBM; append takes 76 us, read
// 68 (f16) and 63 (bf16).  What bounds append is the number of instructions a
// channel (two thirds of the issue slots taken), hence the packing below; what
// bounds read is the latency of three loads in a row, hence two heads a thread
// (one: 82, 78 and 79 us).  Few rows take a launch.  A thread owns a group of 16
// channels of a row, 32 contiguous bytes, so a group's maximum needs no exchange
// between threads.  A block is 16 rows of two heads, 4 warps for K and 4 for V
// (a warp with both would run both codes).
#include "q4_attn.cuh"

namespace dfl {

// Scale byte of a group whose largest magnitude is a: the smallest scale
// >= a / 7.5.  a has at most 11 significant bits and a scale 4, so a / 7.5 is
// either exactly a scale or at least 2^-12 (relative) away from every one:
// shrinking the quotient by 2^-20 keeps an exact one from rounding up past
// itself (the quotient below is a product with 1 / 7.5, off by 2^-23) and
// changes no other result.
__device__ __forceinline__ uint32_t q4_scale_code(float a) {
  const float t = a * (float)((1.0 / 7.5) * (1.0 - 1.0 / (1 << 20)));
  if (t >= 9216.f) return 0xE1;                    // 9216, the largest
  if (t < 6.103515625e-05f) {                      // below 2^-14: multiples of 2^-17
    const int m = (int)ceilf(t * 131072.f);
    return m < 1 ? 1 : m;
  }
  const uint32_t up = (__float_as_uint(t) + 0xFFFFFu) >> 20;   // exponent and 3 mantissa bits, rounded up
  return up - ((127 - 15) << 3);
}

// largest magnitude of 16 values, NaN if one is NaN
template <bool BF16>
__device__ __forceinline__ float group_max(const uint32_t (&u)[8]) {
  uint32_t m = u[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    if (BF16)
      asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(u[i] & 0x7fff7fffu));
    else
      asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(u[i] & 0x7fff7fffu));
  }
  const float lo = BF16 ? __uint_as_float(m << 16) : __half2float(__ushort_as_half((unsigned short)m));
  const float hi = BF16 ? __uint_as_float(m & 0xffff0000u) : __half2float(__ushort_as_half((unsigned short)(m >> 16)));
  float a;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(lo), "f"(hi));
  return a;
}

template <bool BF16>
__global__ void __launch_bounds__(256) q4_append_kernel(const Q4AppendParams p) {
  const int t = threadIdx.x, g = t & 7, which = t >> 7;
  const int row = blockIdx.x * 16 + (t >> 3 & 15), h0 = 2 * blockIdx.y;
  griddep_wait();
  griddep_launch_dependents();
  int slot = row < p.T ? __ldg(p.slots + row) : -1;
  if (slot >= p.num_slots) slot = -1;
  const int other_slot = __shfl_xor_sync(0xffffffffu, slot, 8);   // of the row beside it
  // two heads a thread, their loads on the way together
  uint4 w[2][2] = {};
  if (slot >= 0) {
    const char* src = static_cast<const char*>(which ? p.v : p.k) +
                      2 * ((which ? row * p.v_row + h0 * p.v_head : row * p.k_row + h0 * p.k_head) + 16 * g);
    w[0][0] = ldg_stream(src);
    w[0][1] = ldg_stream(src + 16);
    if (h0 + 1 < p.nkv) {
      src += 2 * (which ? p.v_head : p.k_head);
      w[1][0] = ldg_stream(src);
      w[1][1] = ldg_stream(src + 16);
    }
  }
#pragma unroll
  for (int hh = 0; hh < 2; ++hh) {
    const int h = h0 + hh;
    if (h >= p.nkv) break;
    uint32_t u[8] = {w[hh][0].x, w[hh][0].y, w[hh][0].z, w[hh][0].w, w[hh][1].x, w[hh][1].y, w[hh][1].z, w[hh][1].w};
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (BF16) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
    float a = group_max<BF16>(u);
    if (!(a < INFINITY)) {   // NaN counts as 0 and is stored as 0
      if (p.status) atomicOr(p.status, kPagedNonFinite);
      a = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = x[i] != x[i] ? 0.f : x[i];
        a = fmaxf(a, fabsf(x[i]));
      }
    }
    const uint32_t code = q4_scale_code(a);
    // x / s rounded to nearest, halves away from zero: half-way cases are exact
    // quotients and every other one is at least 2^-12 from a half, so a factor
    // 1 + 2^-16 (2^-13 at 7.5; the reciprocal is off by 2^-22) carries halves
    // outwards and changes nothing else.
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(__half2float(__ushort_as_half((unsigned short)(code << 7)))));
    inv *= 1.f + 1.f / 65536;
    if (a * inv >= 7.5f) {   // the maximum itself would round to 8
      const float most = 7.25f / inv;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fminf(fmaxf(x[i], -most), most);
    }
    // The sum with 1.5 * 2^23 + 8 rounds, and leaves u = q + 8 in the lowest bits;
    // shifting and adding such numbers packs them (the rest stays above bit 16).
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = fmaf(x[i], inv, 12582920.f);
    auto pack4 = [&](int a0, int a1, int a2, int a3) {
      return __float_as_uint(x[a0]) + (__float_as_uint(x[a1]) << 4) + (__float_as_uint(x[a2]) << 8) +
             (__float_as_uint(x[a3]) << 12);
    };
    const int bits = p.page_shift - 4;
    uint8_t* blk = p.pool + ((((size_t)(slot >> p.page_shift) * p.nkv + h) << bits) +
                             (slot / kQ4Rows & ((1 << bits) - 1))) * kQ4Block;
    const int rr = slot & 15;
    if (which == 0) {
      if (slot < 0) continue;
      // channel 2n of a word in its lower half, 2n + 1 in the upper
      *reinterpret_cast<uint2*>(blk + q4_k_piece(rr, g >> 1) + (g & 1) * 8) =
          make_uint2(__byte_perm(pack4(0, 2, 4, 6), pack4(1, 3, 5, 7), 0x5410),
                     __byte_perm(pack4(8, 10, 12, 14), pack4(9, 11, 13, 15), 0x5410));
      blk[kQ4KS + rr * 8 + g] = (uint8_t)code;
    } else {
      const uint32_t h01 = __byte_perm(pack4(0, 1, 2, 3), pack4(4, 5, 6, 7), 0x5410);
      const uint32_t h23 = __byte_perm(pack4(8, 9, 10, 11), pack4(12, 13, 14, 15), 0x5410);
      const uint32_t o01 = __shfl_xor_sync(0xffffffffu, h01, 8), o23 = __shfl_xor_sync(0xffffffffu, h23, 8);
      if (slot < 0) continue;
      uint8_t* piece = blk + kQ4V + q4_v_piece(rr >> 1, g);
      const bool first = !(rr & 1);
      if (other_slot == (slot ^ 1) && first == !(t & 8)) {
        // both rows of the piece are here: half of it each
        if (first)
          *reinterpret_cast<uint2*>(piece) = make_uint2(__byte_perm(h01, o01, 0x5410), __byte_perm(h01, o01, 0x7632));
        else
          *reinterpret_cast<uint2*>(piece + 8) = make_uint2(__byte_perm(o23, h23, 0x5410), __byte_perm(o23, h23, 0x7632));
      } else {
        uint16_t* d = reinterpret_cast<uint16_t*>(piece) + (rr & 1);
        d[0] = (uint16_t)h01;
        d[2] = (uint16_t)(h01 >> 16);
        d[4] = (uint16_t)h23;
        d[6] = (uint16_t)(h23 >> 16);
      }
      blk[kQ4VS + g * 16 + rr] = (uint8_t)code;
    }
  }
}

template <bool BF16>
__global__ void __launch_bounds__(256) q4_read_kernel(const Q4ReadParams p) {
  const int t = threadIdx.x, g = t & 7, which = t >> 7;
  const int row = blockIdx.x * 16 + (t >> 3 & 15), h0 = 2 * blockIdx.y;
  griddep_wait();
  griddep_launch_dependents();
  if (row >= p.T) return;
  const int slot = __ldg(p.slots + row);
  const bool there = slot >= 0 && slot < p.num_slots;
  const int bits = p.page_shift - 4, rr = slot & 15;
  uint4 w[2] = {};
  uint32_t code[2] = {0, 0};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (!there || h0 + x >= p.nkv) continue;
    const uint8_t* blk = p.pool + ((((size_t)(slot >> p.page_shift) * p.nkv + h0 + x) << bits) +
                                   (slot / kQ4Rows & ((1 << bits) - 1))) * kQ4Block;
    code[x] = __ldg(blk + (which ? kQ4VS + g * 16 + rr : kQ4KS + rr * 8 + g));
    if (which == 0) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(blk + q4_k_piece(rr, g >> 1) + (g & 1) * 8));
      w[x].x = v.x;
      w[x].y = v.y;
    } else {
      w[x] = __ldg(reinterpret_cast<const uint4*>(blk + kQ4V + q4_v_piece(rr >> 1, g)));
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    if (h0 + x >= p.nkv) break;
    uint32_t o[8];   // (a slot outside the pool: scale 0 and codes 0)
    const uint32_t s = scale_pair(code[x] | code[x] << 8), ns = scale_shift(s);
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t ww = i ? w[x].y : w[x].x;
        o[4 * i] = dequant<0>(ww, s, ns);
        o[4 * i + 1] = dequant<1>(ww, s, ns);
        o[4 * i + 2] = dequant<2>(ww, s, ns);
        o[4 * i + 3] = dequant<3>(ww, s, ns);
      }
    } else {
      const uint32_t ww[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t hw = (rr & 1) ? ww[i] >> 16 : ww[i] & 0xffffu;
        const uint32_t both = hw | hw << 12;   // channels 4i and 4i + 1 (4i + 2 and 4i + 3) one half apart
        o[2 * i] = dequant<0>(both, s, ns);
        o[2 * i + 1] = dequant<2>(both, s, ns);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = there ? hmul2_u(o[i], 0x4C004C00u) : 0u;   // times 16
      if (BF16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[i]));
        o[i] = pack_bf16x2(f.x, f.y);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(which ? p.v : p.k) + 2 * (((size_t)row * p.nkv + h0 + x) * 128 + 16 * g));
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

cudaError_t q4_append_launch(const Q4AppendParams& p, cudaStream_t st) {
  if (p.T < 1 || p.nkv < 1 || p.nkv > 65535) return cudaErrorInvalidValue;
  const dim3 grid((p.T + 15) / 16, (p.nkv + 1) / 2);
  return launch_pdl(p.bf16 ? q4_append_kernel<true> : q4_append_kernel<false>, grid, dim3(256), 0, st, p);
}

cudaError_t q4_read_launch(const Q4ReadParams& p, cudaStream_t st) {
  if (p.T < 1 || p.nkv < 1 || p.nkv > 65535) return cudaErrorInvalidValue;
  const dim3 grid((p.T + 15) / 16, (p.nkv + 1) / 2);
  return launch_pdl(p.bf16 ? q4_read_kernel<true> : q4_read_kernel<false>, grid, dim3(256), 0, st, p);
}

}  // namespace dfl
