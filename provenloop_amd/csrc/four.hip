// 4-bit weights: quantizing, laying out given codes, and their values.
//
// Quantizing a group of columns of a row, sums and quotients in float:
//   without zeros  scale = T(max |w| / 7),                 code = clamp(rint(w / scale), -7, 7) + 8
//   with zeros     scale = T((max(w, 0) - min(w, 0)) / 15), zero = clamp(rint(-min(w, 0) / scale), 0, 15),
//                  code = clamp(rint(w / scale) + zero, 0, 15)
// with the scale rounded to the weights' type T first, so that the codes are the
// nearest to what they will stand for. Codes do not depend on the quotient's own
// rounding: a tie is (n + 1/2) scale, 4 bits times at most 11, and a value of T
// that is not on it is off by more than 2^-16 of it.
//
// All three move bytes (2 a value, 1 a given code, half a byte of ours), a
// wavefront for 16 rows with 8 columns of a row in each lane, the layout's own
// (mixture_rules.h): 8 matrices of 3584 x 1536 in groups of 128 columns take 22.4 us to
// 4 bits (4.9 TB/s; in groups of 64 with zeros 25), 22.0 back, and 15.9 from given codes
// (4.2 TB/s). Quantizing gives a group of columns of 16 rows to one wavefront, so long
// groups leave CUs without work (3584 x 3584: 8.4 us for 128 columns, 23 for 1024, 70
// for 4096).
#include "four_device.h"

namespace {

// A scale as it is stored: the values of a group whose scale is not a number the
// products can use (an infinity, NaN, in bf16 above 2^120) are NaN.
template <class T>
__device__ inline T stored_scale(T s) {
  const bool fine = std::is_same<T, bf16_t>::value ? fabsf((float)s) <= 0x1p120f : is_finite(s);
  return fine ? s : (T)NAN;
}

__device__ inline float over_row(float v, bool most) {
#pragma unroll
  for (int d = 16; d < 64; d *= 2) {
    const float o = __shfl_xor(v, d);
    v = most ? fmaxf(v, o) : fminf(v, o);
  }
  return v;
}

// Which strip of which matrix a workgroup takes, and its share of what lies along it.
struct Share {
  uint32_t strip, part, parts;
  uint64_t e;
};
__device__ inline Share share_of(const FourRows& a, uint32_t parts) {
  const uint32_t job = blockIdx.x / parts;
  return Share{job % a.four.at.strips, blockIdx.x % parts, parts, job / a.four.at.strips};
}

// Codes of 8 values of a group, as their word. rint(v / s), ties to even, for v and s
// of T with a quotient below 16: v / s is a tie, n + 1/2, or off any by more than
// 2^-13 (both have 11 bits at most), and v times the rounded reciprocal is off by
// less than 2^-18; rounded to a multiple of 2^-14 it is the tie, or on its own side
// of it. That and the conversion of 8 values into bytes are 50 instructions, quotients
// and shifts were 130.
template <bool ZEROS>
struct Coder {
  float per, scale, zero;
  bool small;  // the reciprocal would be infinite
  __device__ inline Coder(float s, float z) : per(0x1p14f / s), scale(s), zero(z), small(s < 0x1p-100f) {}
  template <class V>
  __device__ inline uint32_t word(const V& v, bool slow) const {
    uint32_t even = 0, odd = 0;  // a byte a code: columns 0, 4, 1, 5 and 2, 6, 3, 7
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = rintf(slow ? (float)v[i] / scale * 0x1p14f : (float)v[i] * per);
      // 8 is even: rounding to a byte comes out the same with it added before
      float c = ZEROS ? rintf(t * 0x1p-14f) + zero : fmaf(t, 0x1p-14f, 8.0f);
      c = __builtin_amdgcn_fmed3f(c, ZEROS ? 0.0f : 1.0f, 15.0f);
      uint32_t& w = i / 2 % 2 ? odd : even;
      w = __builtin_amdgcn_cvt_pk_u8_f32(c, i % 2 * 2 + i / 4, w);
    }
    return even | odd << 4;
  }
};

// A wavefront a group of columns of 16 rows. KEEP: steps of 32 columns whose
// values stay in registers; longer groups are read again for their codes.
template <class T, int KEEP, bool ZEROS>
__global__ void __launch_bounds__(256) quantize4_kernel(FourRows a, uint32_t parts) {
  typedef __attribute__((ext_vector_type(8))) uint16_t u16x8;
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const Share m = share_of(a, parts);
  const uint32_t row = m.strip * 16 + lane % 16;
  const T* in = (const T*)a.in + (int64_t)m.e * a.lde + (int64_t)min(row, a.rows - 1) * a.ld;
  uint8_t* out = (uint8_t*)a.four.codes + m.e * f.codes() + (uint64_t)m.strip * f.blocks * 512 + lane * 8;
  for (uint32_t g = m.part * 4 + (threadIdx.x >> 6); g < f.groups; g += parts * 4) {
    const uint32_t k0 = g << f.shift;
    const uint32_t k1 = (uint32_t)min((uint64_t)k0 + (1ull << f.shift), (uint64_t)f.blocks * 64), steps = (k1 - k0) / 32;
    auto fetch = [&](uint32_t step) __attribute__((always_inline)) {
      const uint32_t k = k0 + step * 32 + lane / 16 * 8;
      const bool in_row = row < a.rows && k < a.cols;
      return load8<T>(in_row ? in + k : (const T*)&mix_zero16, in_row ? (int64_t)a.cols - k : 0);
    };
    vec8<T> kept[KEEP];
    // without zeros, the largest magnitude as its bits, which order like it; NaN and infinity are above all
    u16x8 size = 0;
    float low = 0, high = 0;
    bool bad = false;
    auto look = [&](const vec8<T>& v) __attribute__((always_inline)) {
      if constexpr (!ZEROS) {
        size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x8, v) & (uint16_t)0x7fff);
      } else {
        bad |= !all_finite<T>(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          low = fminf(low, (float)v[i]);
          high = fmaxf(high, (float)v[i]);
        }
      }
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i < (int)steps) kept[i] = fetch(i);
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i < (int)steps) look(kept[i]);
    for (uint32_t i = KEEP; i < steps; ++i) look(fetch(i));
    if constexpr (!ZEROS) {
      uint16_t most = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = most > size[i] ? most : size[i];
      bad = most >= exponent_bits<T>();
      high = (float)__builtin_bit_cast(T, bad ? (uint16_t)0 : most);
    } else {
      low = over_row(low, false);
    }
    high = over_row(high, true);
    bad = over_row(bad ? 1.0f : 0.0f, true) != 0;
    const T scale = stored_scale((T)(bad ? NAN : ZEROS ? (high - low) / 15.0f : high / 7.0f));
    const float by = (float)scale > 0 ? (float)scale : 1.0f;
    const bool number = (float)scale == (float)scale;
    const float zero = ZEROS && number ? fminf(rintf(-low / by), 15.0f) : 8.0f;
    const Coder<ZEROS> coder(by, zero);
    const bool slow = __any(coder.small);
    auto code = [&](const vec8<T>& v, uint32_t step) __attribute__((always_inline)) {
      const uint32_t k = k0 + step * 32;
      const uint32_t w = slow ? coder.word(v, coder.small) : coder.word(v, false);
      *(uint32_t*)(out + (uint64_t)(k / 64) * 512 + k / 32 % 2 * 4) = number ? w : 0x88888888u;
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i < (int)steps) code(kept[i], i);
    for (uint32_t i = KEEP; i < steps; ++i) code(fetch(i), i);
    if (lane < 16) {
      const uint64_t at = m.e * f.scales() + (uint64_t)g * f.strips * 16 + row;
      ((T*)a.four.scales)[at] = row < a.rows ? scale : (T)0.0f;
      if (ZEROS) ((uint8_t*)a.four.zeros)[at] = (uint8_t)zero;
    }
  }
}

// A wavefront a block of 16 rows by 64 columns: codes, and the scales and zeros
// of the groups that begin there.
template <class T>
__global__ void __launch_bounds__(256) pack4_kernel(FourRows a, uint32_t parts) {
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const Share m = share_of(a, parts);
  const uint32_t row = m.strip * 16 + lane % 16;
  const uint8_t* in = (const uint8_t*)a.in + (int64_t)m.e * a.lde + (int64_t)min(row, a.rows - 1) * a.ld;
  uint8_t* out = (uint8_t*)a.four.codes + m.e * f.codes() + (uint64_t)m.strip * f.blocks * 512 + lane * 8;
  for (uint32_t block = m.part * 4 + (threadIdx.x >> 6); block < f.blocks; block += parts * 4) {
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t k = block * 64 + h * 32 + lane / 16 * 8;
      uint32_t c[8];
      uint64_t w = 0x0808080808080808ull;
      const bool whole = row < a.rows && k + 8 <= a.cols;
      if (whole) {
        __builtin_memcpy(&w, in + k, 8);
      } else if (a.four.zeros && row < a.rows && k >> f.shift < a.scale_cols) {
        // behind the last column the value 0: another one's multiple of the scale may be infinite
        w = 0x0101010101010101ull * (a.zeros[(m.e * a.rows + row) * a.scale_cols + (k >> f.shift)] & 15);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = (uint32_t)(w >> (8 * i)) & 15;
        if (!whole && row < a.rows && k + i < a.cols) c[i] = in[k + i] & 15;
      }
      q[h] = four_word(c);
    }
    *(uint2*)(out + (uint64_t)block * 512) = uint2{q[0], q[1]};
    // group number h of the block, if it begins here
    const uint32_t h = lane / 16, k = block * 64 + h * 32, g = k >> f.shift;
    if (h < 2 && k == g << f.shift) {
      const bool in_rows = row < a.rows && g < a.scale_cols;
      const uint64_t from = (m.e * a.rows + row) * a.scale_cols + g;
      const uint64_t to = m.e * f.scales() + (uint64_t)g * f.strips * 16 + row;
      ((T*)a.four.scales)[to] = in_rows ? stored_scale(((const T*)a.scales)[from]) : (T)0.0f;
      if (a.four.zeros) ((uint8_t*)a.four.zeros)[to] = in_rows ? a.zeros[from] & 15 : 8;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) dequantize4_kernel(FourRows a, uint32_t parts) {
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const Share m = share_of(a, parts);
  const uint32_t row = m.strip * 16 + lane % 16;
  const bool wide = ((uintptr_t)a.out & 15) == 0 && a.ld % 8 == 0 && a.lde % 8 == 0;
  const uint8_t* in = a.four.codes + m.e * f.codes() + (uint64_t)m.strip * f.blocks * 512 + lane * 8;
  const uint64_t scales = m.e * f.scales() + row, per = (uint64_t)f.strips * 16;
  T* out = (T*)a.out + (int64_t)m.e * a.lde + (int64_t)row * a.ld;
  for (uint32_t block = m.part * 4 + (threadIdx.x >> 6); block < f.blocks; block += parts * 4) {
    const uint2 q = *(const uint2*)(in + (uint64_t)block * 512);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t k = block * 64 + h * 32 + lane / 16 * 8;
      const uint64_t at = scales + (k >> f.shift) * per;
      const FourScale<T> s(((const T*)a.four.scales)[at], a.four.zeros ? a.four.zeros[at] : 8);
      vec8<T> v = four_values(h ? q.y : q.x, s);
      if (row >= a.rows || k >= a.out_cols) continue;
      if (k + 8 > a.cols)
        for (uint32_t i = 0; i < 8; ++i) v[i] = k + i < a.cols ? v[i] : (T)0.0f;
      if (wide && k + 8 <= a.out_cols) *(vec8<T>*)(out + k) = v;
      else
        for (uint32_t i = 0; i < 8; ++i)
          if (k + i < a.out_cols) out[k + i] = v[i];
    }
  }
}

// Workgroups that share a strip's n blocks or groups, four of them at a time: enough
// for 4096 in all, as far as there is that much to share.
uint32_t parts_of(const FourRows& a, uint32_t n) {
  const uint64_t strips = (uint64_t)a.E * a.four.at.strips, most = th::ceil_div(n, 4), want = th::ceil_div(4096, strips);
  return (uint32_t)(want < most ? want : most);
}
template <auto Kernel>
hipError_t go(const FourRows& a, uint32_t n, hipStream_t s) {
  const uint32_t parts = parts_of(a, n);
  return launch<Kernel>((uint64_t)a.E * a.four.at.strips * parts, 256, 0, s, a, parts);
}

template <class T, bool ZEROS>
hipError_t quantize(const FourRows& a, hipStream_t s) {
  const th::FourLayout& f = a.four.at;
  switch (f.shift) {
    case 5: return go<quantize4_kernel<T, 1, ZEROS>>(a, f.groups, s);
    case 6: return go<quantize4_kernel<T, 2, ZEROS>>(a, f.groups, s);
    default: return go<quantize4_kernel<T, 4, ZEROS>>(a, f.groups, s);
  }
}

}  // namespace

hipError_t launch_quantize4(MixType type, const FourRows& a, hipStream_t s) {
  if (a.four.zeros) return type == MIX_BF16 ? quantize<bf16_t, true>(a, s) : quantize<f16_t, true>(a, s);
  return type == MIX_BF16 ? quantize<bf16_t, false>(a, s) : quantize<f16_t, false>(a, s);
}

hipError_t launch_pack4(MixType type, const FourRows& a, hipStream_t s) {
  return type == MIX_BF16 ? go<pack4_kernel<bf16_t>>(a, a.four.at.blocks, s) : go<pack4_kernel<f16_t>>(a, a.four.at.blocks, s);
}

hipError_t launch_dequantize4(MixType type, const FourRows& a, hipStream_t s) {
  return type == MIX_BF16 ? go<dequantize4_kernel<bf16_t>>(a, a.four.at.blocks, s)
                          : go<dequantize4_kernel<f16_t>>(a, a.four.at.blocks, s);
}
