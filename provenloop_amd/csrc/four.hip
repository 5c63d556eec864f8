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
// (mixture_rules.h).
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

// A wavefront a group of columns of 16 rows. KEEP: steps of 32 columns whose
// values stay in registers; longer groups are read again for their codes.
template <class T, int KEEP>
__global__ void __launch_bounds__(256) quantize4_kernel(FourRows a) {
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const uint64_t jobs = (uint64_t)a.E * f.strips * f.groups;
  for (uint64_t job = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (uint64_t)gridDim.x * 4) {
    const uint32_t g = job % f.groups, strip = job / f.groups % f.strips, e = job / f.groups / f.strips;
    const uint32_t row = strip * 16 + lane % 16, k0 = g << f.shift;
    const uint32_t k1 = (uint32_t)min((uint64_t)k0 + (1ull << f.shift), (uint64_t)f.blocks * 64), steps = (k1 - k0) / 32;
    const T* in = (const T*)a.in + (int64_t)e * a.lde + (int64_t)min(row, a.rows - 1) * a.ld;
    auto fetch = [&](uint32_t step) __attribute__((always_inline)) {
      const uint32_t k = k0 + step * 32 + lane / 16 * 8;
      const bool in_row = row < a.rows && k < a.cols;
      return load8<T>(in_row ? in + k : (const T*)&mix_zero16, in_row ? (int64_t)a.cols - k : 0);
    };
    vec8<T> kept[KEEP];
    float low = 0, high = 0;
    bool bad = false;
    auto look = [&](const vec8<T>& v) __attribute__((always_inline)) {
      bad |= !all_finite<T>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        low = fminf(low, (float)v[i]);
        high = fmaxf(high, (float)v[i]);
      }
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i < (int)steps) {
        kept[i] = fetch(i);
        look(kept[i]);
      }
    for (uint32_t i = KEEP; i < steps; ++i) look(fetch(i));
    low = over_row(low, false);
    high = over_row(high, true);
    bad = over_row(bad ? 1.0f : 0.0f, true) != 0;
    const bool zeros = a.four.zeros != nullptr;
    const T scale = stored_scale((T)(bad ? NAN : zeros ? (high - low) / 15.0f : fmaxf(-low, high) / 7.0f));
    const float by = (float)scale > 0 ? (float)scale : 1.0f;
    const bool number = (float)scale == (float)scale;
    const float zero = zeros && number ? fminf(rintf(-low / by), 15.0f) : 8.0f, least = zeros ? 0.0f : 1.0f;
    auto code = [&](const vec8<T>& v, uint32_t step) __attribute__((always_inline)) {
      uint32_t c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        c[i] = number ? (uint32_t)fminf(fmaxf(rintf((float)v[i] / by) + zero, least), 15.0f) : 8;
      const uint32_t k = k0 + step * 32;
      uint8_t* out = (uint8_t*)a.four.codes + e * f.codes() + ((uint64_t)strip * f.blocks + k / 64) * 512;
      *(uint32_t*)(out + lane * 8 + k / 32 % 2 * 4) = four_word(c);
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (i < (int)steps) code(kept[i], i);
    for (uint32_t i = KEEP; i < steps; ++i) code(fetch(i), i);
    if (lane < 16) {
      const uint64_t at = e * f.scales() + (uint64_t)g * f.strips * 16 + row;
      ((T*)a.four.scales)[at] = row < a.rows ? scale : (T)0.0f;
      if (zeros) ((uint8_t*)a.four.zeros)[at] = (uint8_t)zero;
    }
  }
}

// A wavefront a block of 16 rows by 64 columns: codes, and the scales and zeros
// of the groups that begin there.
template <class T>
__global__ void __launch_bounds__(256) pack4_kernel(FourRows a) {
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const uint64_t jobs = (uint64_t)a.E * f.strips * f.blocks;
  for (uint64_t job = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (uint64_t)gridDim.x * 4) {
    const uint32_t block = job % f.blocks, strip = job / f.blocks % f.strips, e = job / f.blocks / f.strips;
    const uint32_t row = strip * 16 + lane % 16;
    const uint8_t* in = (const uint8_t*)a.in + (int64_t)e * a.lde + (int64_t)min(row, a.rows - 1) * a.ld;
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t k = block * 64 + h * 32 + lane / 16 * 8;
      uint32_t c[8];
      uint64_t w = 0x0808080808080808ull;
      const bool whole = row < a.rows && k + 8 <= a.cols;
      if (whole) __builtin_memcpy(&w, in + k, 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = (uint32_t)(w >> (8 * i)) & 15;
        if (!whole && row < a.rows && k + i < a.cols) c[i] = in[k + i] & 15;
      }
      q[h] = four_word(c);
    }
    *(uint2*)((uint8_t*)a.four.codes + job * 512 + lane * 8) = uint2{q[0], q[1]};
    // group number h of the block, if it begins here
    const uint32_t h = lane / 16, k = block * 64 + h * 32, g = k >> f.shift;
    if (h < 2 && k == g << f.shift) {
      const bool in_rows = row < a.rows && g < a.scale_cols;
      const uint64_t from = ((uint64_t)e * a.rows + row) * a.scale_cols + g;
      const uint64_t to = e * f.scales() + (uint64_t)g * f.strips * 16 + row;
      ((T*)a.four.scales)[to] = in_rows ? stored_scale(((const T*)a.scales)[from]) : (T)0.0f;
      if (a.four.zeros) ((uint8_t*)a.four.zeros)[to] = in_rows ? a.zeros[from] & 15 : 8;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(256) dequantize4_kernel(FourRows a) {
  const uint32_t lane = threadIdx.x & 63;
  const th::FourLayout f = a.four.at;
  const uint64_t jobs = (uint64_t)a.E * f.strips * f.blocks;
  const bool wide = ((uintptr_t)a.out & 15) == 0 && a.ld % 8 == 0 && a.lde % 8 == 0;
  for (uint64_t job = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (uint64_t)gridDim.x * 4) {
    const uint32_t block = job % f.blocks, strip = job / f.blocks % f.strips, e = job / f.blocks / f.strips;
    const uint32_t row = strip * 16 + lane % 16;
    const uint2 q = *(const uint2*)(a.four.codes + job * 512 + lane * 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t k = block * 64 + h * 32 + lane / 16 * 8;
      const uint64_t at = e * f.scales() + (uint64_t)(k >> f.shift) * f.strips * 16 + row;
      const FourScale<T> s(((const T*)a.four.scales)[at], a.four.zeros ? a.four.zeros[at] : 8);
      vec8<T> v = four_values(h ? q.y : q.x, s);
      if (row >= a.rows || k >= a.out_cols) continue;
      T* out = (T*)a.out + (int64_t)e * a.lde + (int64_t)row * a.ld + k;
      if (k + 8 > a.cols)
        for (uint32_t i = 0; i < 8; ++i) v[i] = k + i < a.cols ? v[i] : (T)0.0f;
      if (wide && k + 8 <= a.out_cols) *(vec8<T>*)out = v;
      else
        for (uint32_t i = 0; i < 8; ++i)
          if (k + i < a.out_cols) out[i] = v[i];
    }
  }
}

uint32_t blocks_for(uint64_t jobs) { return th::loop_blocks(th::ceil_div(jobs, 4)); }

template <class T>
hipError_t quantize(const FourRows& a, hipStream_t s) {
  const th::FourLayout& f = a.four.at;
  const uint32_t blocks = blocks_for((uint64_t)a.E * f.strips * f.groups);
  switch (f.shift) {
    case 5: return launch<quantize4_kernel<T, 1>>(blocks, 256, 0, s, a);
    case 6: return launch<quantize4_kernel<T, 2>>(blocks, 256, 0, s, a);
    default: return launch<quantize4_kernel<T, 4>>(blocks, 256, 0, s, a);
  }
}

}  // namespace

hipError_t launch_quantize4(MixType type, const FourRows& a, hipStream_t s) {
  return type == MIX_BF16 ? quantize<bf16_t>(a, s) : quantize<f16_t>(a, s);
}

hipError_t launch_pack4(MixType type, const FourRows& a, hipStream_t s) {
  const uint32_t blocks = blocks_for((uint64_t)a.E * a.four.at.strips * a.four.at.blocks);
  return type == MIX_BF16 ? launch<pack4_kernel<bf16_t>>(blocks, 256, 0, s, a)
                          : launch<pack4_kernel<f16_t>>(blocks, 256, 0, s, a);
}

hipError_t launch_dequantize4(MixType type, const FourRows& a, hipStream_t s) {
  const uint32_t blocks = blocks_for((uint64_t)a.E * a.four.at.strips * a.four.at.blocks);
  return type == MIX_BF16 ? launch<dequantize4_kernel<bf16_t>>(blocks, 256, 0, s, a)
                          : launch<dequantize4_kernel<f16_t>>(blocks, 256, 0, s, a);
}
