// Rules on sizes of the plain mixture-of-adapters operators, apart from HIP so
// that a host program can evaluate them (tests/test_mixture_rules.py).
#pragma once
#include <stddef.h>
#include <stdint.h>

namespace th {

constexpr uint32_t MIX_MAX_EXPERTS = 1024;  // the slot counters of a workgroup: 16 wavefronts x 1025 words of LDS
constexpr uint32_t MIX_MAX_CHOICES = 32;
constexpr uint32_t MIX_MAX_RANK = 128;      // eight 16-row tiles of an adapter held by one workgroup

constexpr uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// A launch has fewer than 2^32 threads along each axis; the runtime takes more
// with their number wrapped round.
constexpr bool launchable(uint64_t blocks, uint32_t threads) { return blocks < (1ull << 32) / threads; }
// What make() gives, asked for once per Kernel: kernels are functions, and many
// of them have one type.
template <auto Kernel, class Make>
auto once_for(Make make) {
  static const auto made = make();
  return made;
}
// Workgroups of a kernel whose workgroups each take every so-many-th piece of
// work: 2^20 fill the GPU many times over.
constexpr uint32_t loop_blocks(uint64_t pieces) { return (uint32_t)(pieces < 1u << 20 ? pieces : 1u << 20); }

// Tokens whose (token, choice) slots one workgroup of 1024 threads groups: 1024
// to 4096 slots, as few as give a workgroup to each of the 256 CUs, and more
// where there would be more than 1024 workgroups, each of which adds up the
// others' counts. One workgroup alone needs no second launch, so up to 2048
// slots stay whole.
constexpr uint64_t group_chunk_tokens(uint64_t tokens, uint32_t k) {
  const uint64_t slots = tokens * k;
  uint64_t chunk = slots <= 2048 ? 2048 : ceil_div(slots, 256);
  chunk = chunk < 1024 ? 1024 : chunk > 4096 ? 4096 : chunk;
  if (chunk < ceil_div(slots, 1024)) chunk = ceil_div(slots, 1024);
  const uint64_t t = chunk / k;
  return t ? t : 1;
}
constexpr uint64_t group_chunks(uint64_t tokens, uint32_t k) {
  return tokens ? ceil_div(tokens, group_chunk_tokens(tokens, k)) : 1;
}

// Slots of one partial sum of a low-rank gradient, and how many there are at
// most: spans of 256 to 2048 slots, doubled while the launch has workgroups to
// spare (128 columns each).
constexpr uint32_t lowrank_span(uint64_t slots, uint32_t cols) {
  uint32_t span = 256;
  while (span < 2048 && ceil_div(slots, span * 2) * ceil_div(cols, 128) >= 1024) span *= 2;
  return span;
}
constexpr uint64_t lowrank_spans(uint64_t slots, uint32_t E, uint32_t span) {
  return slots / span + (E < slots ? E : slots);
}

// Products of few output tiles (narrow.hip). 16 x 16 tiles take 8 wavefronts,
// two workgroups a CU, while those are all there at once, and 4, five a CU, from
// 512 on (8192 slots of 8 groups by 16 columns of 1536 steps: 521 tiles, 9.1 us
// and 11.9 with 8). The tile: 16 rows where groups
// have no more, or the output no more columns (8192 x 16 x 1536: 5.9 us, 6.1
// with 32 rows), else 32; 32 columns once there are enough workgroups (32 x 3584
// x 3584: 6.7 us with 16 columns, 7.7 with 32; 250 x 1536 x 1536: 9.0 and 6.7).
enum NarrowTile { NARROW_16x16, NARROW_32x16, NARROW_32x32, NARROW_16x16_MANY };
constexpr NarrowTile narrow_tile(uint64_t rows, uint32_t n, uint32_t groups) {
  const uint64_t each = ceil_div(rows, groups);
  if (each <= 16 || n <= 16) return groups * ceil_div(each, 16) * ceil_div(n, 16) < 512 ? NARROW_16x16 : NARROW_16x16_MANY;
  return groups * ceil_div(each, 32) * ceil_div(n, 32) < 192 ? NARROW_32x16 : NARROW_32x32;
}
// Whether a product is one of those: up to 1024 tiles of 32 x 32, about what the
// time of one round of large tiles pays for (narrow / wide in us: 256 columns of
// 1536 steps, 2048 rows 12.6 / 21.1, 4096 rows 22.9 / 21.4; 1536 of 1536, 512
// rows 15.7 / 21.5, 1024 rows 25.9 / 22.4; 3584 of 3584, 256 rows 26 / 42, 512
// rows 45 / 43; 4096 of 512, 128 rows 7.3 / 11.4, 256 rows 12.3 / 11.7). Groups of
// up to 16 rows are weights to be read, which small tiles do faster if the
// contraction is long (8 groups of 8 rows: 3584 of 3584 38 / 54, 4096 of 512
// 20 / 13).
constexpr bool narrow_product(uint64_t rows, uint32_t n, uint32_t k, uint32_t groups) {
  const uint64_t each = ceil_div(rows, groups);
  if (each <= 16) return k >= 1024 || groups * ceil_div(n, 16) <= 1024;
  return groups * ceil_div(each, 32) * ceil_div(n, 32) <= 1024;
}
// The wide products' tile: 256 x 256 or 256 x 128. A CU holds one workgroup of
// either, and a square tile takes 1.75 times as long as the other (1.72 and
// 0.97 us per 64 steps at 8192 x 8192 x 8192, in turn in short series), so it is
// better where the number of rounds over the 256 CUs allows it: 8192 x 3584 x
// 3584 takes 204 us with squares and 249 with halves, 4096 x 1536 x 1536 36 and
// 24.5.
constexpr bool wide_square(uint64_t rows, uint32_t n, uint32_t groups) {
  const uint64_t m = groups * ceil_div(ceil_div(rows, groups), 256);
  return ceil_div(m * ceil_div(n, 256), 256) * 7 <= ceil_div(m * ceil_div(n, 128), 256) * 4;
}
// Whether operands that do not start on 16 bytes, or are no multiple of 8 wide,
// are copied to ones that are (as they are / copied, in us a call: 1 row of 3585
// -> 3584 30 / 27, 16 rows 42 / 27; 1537 -> 1536, 1 row 17 / 14, 32 rows 27 / 17;
// 203 -> 515, 1 row 8.6 / 12.1, 32 rows 10.3 / 12.4; 1427 rows of 1389 -> 544
// 82 / 41): a short contraction of few rows does not pay for the launch.
constexpr bool pad_operands(uint64_t rows, uint32_t k) { return rows > 32 || k >= 1024; }
// The workgroups that make such a copy, 2048 values at a time.
constexpr uint32_t pad_blocks(uint64_t rows, uint32_t E, uint32_t cols) {
  return loop_blocks(ceil_div(rows * E * ceil_div(cols, 8), 256));
}
// Slots whose adapters a workgroup of the low-rank product looks through by
// itself, which saves the launch that would group them.
constexpr uint32_t NARROW_SCAN_SLOTS = 2048;

}  // namespace th
