// Rows into and out of the paged 4-bit cache (layout and numbers: q4.cuh).
//
// Both directions stream: 2 bytes a channel on one side, 9/16 on the other, a
// maximum and a rounding between, so HBM bounds them (and a launch's latency
// for the few rows of a decode step).  One thread owns one group of 16
// channels of one row and head, 32 contiguous bytes, so a group's maximum
// needs no exchange between threads.
#include "q4.cuh"

namespace dfl {

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& w, float* x) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF16) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

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

template <bool BF16>
__global__ void __launch_bounds__(256) q4_append_kernel(const Q4AppendParams p) {
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const int g = idx & 7, which = (idx >> 3) & 1;
  const long long rh = idx >> 4;
  const int row = (int)(rh / p.nkv), h = (int)(rh - (long long)row * p.nkv);
  if (row >= p.T) return;
  const int slot = __ldg(p.slots + row);
  if (slot < 0 || slot >= p.num_slots) return;
  const char* src = static_cast<const char*>(which ? p.v : p.k) +
                    2 * ((which ? row * p.v_row + h * p.v_head : row * p.k_row + h * p.k_head) + 16 * g);
  float x[16];
  unpack8<BF16>(ldg_stream(src), x);
  unpack8<BF16>(ldg_stream(src + 16), x + 8);
  float a = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a = fmaxf(a, fabsf(x[i]));                 // fmaxf drops a NaN
    odd |= !(fabsf(x[i]) < INFINITY);
  }
  if (odd && p.status) atomicOr(p.status, kPagedNonFinite);
  const uint32_t code = q4_scale_code(a);
  const float inv = 1.f / __half2float(__ushort_as_half((unsigned short)(code << 7)));
  // Half-way cases are exact quotients; every other one is at least 2^-12 away
  // from a half, so adding 2^-14 beside the 0.5 rounds halves away from zero
  // whatever the reciprocal's last bit, and nothing else differently.
  uint32_t u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float r = fminf(floorf(fmaf(fabsf(x[i]), inv, 0.5f + 1.f / 16384)), 7.f);   // a NaN gives 7: see below
    const int q = x[i] != x[i] ? 0 : (int)r;
    u[i] = x[i] < 0.f ? 8 - q : 8 + q;
  }
  uint8_t* blk = p.pool + q4_block_offset(slot, h, p.nkv, p.page_size);
  const int rr = slot % kQ4Rows;
  if (which == 0) {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[j] = 0;
#pragma unroll
      for (int n = 0; n < 4; ++n) w[j] |= u[8 * j + 2 * n] << (4 * n) | u[8 * j + 2 * n + 1] << (16 + 4 * n);
    }
    *reinterpret_cast<uint2*>(blk + q4_k_piece(rr, g >> 1) + (g & 1) * 8) = make_uint2(w[0], w[1]);
    blk[kQ4KS + rr * 8 + g] = (uint8_t)code;
  } else {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t hw = u[4 * w] | u[4 * w + 1] << 4 | u[4 * w + 2] << 8 | u[4 * w + 3] << 12;
      *reinterpret_cast<uint16_t*>(blk + kQ4V + q4_v_piece(rr >> 1, g) + w * 4 + (rr & 1) * 2) = (uint16_t)hw;
    }
    blk[kQ4VS + g * 16 + rr] = (uint8_t)code;
  }
}

__global__ void __launch_bounds__(256) q4_read_kernel(const Q4ReadParams p) {
  const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
  const int g = idx & 7, which = (idx >> 3) & 1;
  const long long rh = idx >> 4;
  const int row = (int)(rh / p.nkv), h = (int)(rh - (long long)row * p.nkv);
  if (row >= p.T) return;
  const int slot = __ldg(p.slots + row);
  uint32_t o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot >= 0 && slot < p.num_slots) {
    const uint8_t* blk = p.pool + q4_block_offset(slot, h, p.nkv, p.page_size);
    const int rr = slot % kQ4Rows;
    uint32_t u[16], code;
    if (which == 0) {
      const uint2 w = *reinterpret_cast<const uint2*>(blk + q4_k_piece(rr, g >> 1) + (g & 1) * 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) u[i] = ((i < 8 ? w.x : w.y) >> (16 * (i & 1) + 4 * ((i & 7) >> 1))) & 15;
      code = blk[kQ4KS + rr * 8 + g];
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t hw =
            *reinterpret_cast<const uint16_t*>(blk + kQ4V + q4_v_piece(rr >> 1, g) + w * 4 + (rr & 1) * 2);
#pragma unroll
        for (int n = 0; n < 4; ++n) u[4 * w + n] = (hw >> (4 * n)) & 15;
      }
      code = blk[kQ4VS + g * 16 + rr];
    }
    const float s = __half2float(__ushort_as_half((unsigned short)(code << 7)));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lo = ((int)u[2 * i] - 8) * s, hi = ((int)u[2 * i + 1] - 8) * s;
      o[i] = p.bf16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(which ? p.v : p.k) + 2 * (rh * 128 + 16 * g));
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

cudaError_t q4_append_launch(const Q4AppendParams& p, cudaStream_t st) {
  const long long blocks = ((long long)p.T * p.nkv * 16 + 255) / 256;
  if (blocks < 1 || blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (p.bf16)
    q4_append_kernel<true><<<(unsigned)blocks, 256, 0, st>>>(p);
  else
    q4_append_kernel<false><<<(unsigned)blocks, 256, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t q4_read_launch(const Q4ReadParams& p, cudaStream_t st) {
  const long long blocks = ((long long)p.T * p.nkv * 16 + 255) / 256;
  if (blocks < 1 || blocks > INT32_MAX) return cudaErrorInvalidValue;
  q4_read_kernel<<<(unsigned)blocks, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace dfl
