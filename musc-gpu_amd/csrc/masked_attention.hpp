// Softmax attention over the keys that a query may see, for packed images, padded batches,
// prefixes and frames, with an optional cap on the scores and an optional bias by distance:
//
//   score(i, j) = c(scale q_i . k_j) - sum_a slope[head, a] |p_a(i) - p_a(j)|
//   c(s)        = cap tanh(s / cap), or s
//   seen(i, j)  = document(i) == document(j) >= 0 and order(j) <= order(i)
//   out_i       = sum_seen e^(score - max) v_j / sum_seen e^(score - max); zeros if none is seen
//
// One pass over the keys with the running maximum and sum of the softmax.  As in the
// unmasked kernels a wave forms S^T = K Q^T, so that a lane owns one query row and its
// maximum, sum and probabilities stay in its registers; O^T += V^T P^T follows with P in
// place.  16-bit types round P to the storage type for that product, and the sum is of the rounded
// values: half a step of each probability, with which an output is 1.1 to 1.3 times as far from float64 as
// rounding the output alone leaves it, for a product of 8 (fp32: 1) times the rate.  A row is a (token, head of the group) pair: the heads that share a key head are
// neighbouring rows, so K and V are read once for all of them.
//
// Keys come in tiles of 64 (fp32, and workgroups of one wave: 32), staged in LDS straight from
// memory, one tile ahead.  A small summary of the keys (per 32 of them the range of documents and
// orders, made once per batch) sorts a tile, for the rows of a wave, into unseen (skipped without
// reading K or V), seen whole (no mask is evaluated) and mixed (each score is tested).  64 tiles are
// sorted at a time, one per lane.
//
// Rows and keys are shared out three ways:
//   many rows   four waves of 32 rows each on the same tiles.  Row tiles are begun in the order of
//               their work (musc_token_schedule); those of two documents are cut between them, or, with an
//               order of tokens and where all begin at once, long ones are done in parts of their keys
//               (kInParts) that a second kernel joins;
//   few rows    (a new token, a pooling latent) over up to 2048 keys: the waves of one workgroup take
//               every n-th tile of the same rows and join in LDS (kTeams);
//   few rows over more keys: one wave each on a stretch of the keys, four of them on a CU, joined by
//               a second kernel in a fixed order.
//
// What bounds it.  Long rows: a wave and tile of 64 keys costs 512 (heads of 64) or 1024 (128) cycles
// of matrix instructions and about 650 of vector ones (per score: multiply-add, exponential of two
// slots, half a maximum, half a conversion, half a sum), 770 more with a cap (exponential and
// reciprocal), 256 of each kind with a bias over two axes; the two kinds run beside one another
// little.  16 frames of 1024 patches, 16 heads of 128, bf16: 1075 to 1125 us by card, 1.04 to 1.09 PFLOP/s, a
// product of 8192^3 1.14.  8192 tokens, 16 heads of 64, fp16: 336 us, 0.82 PFLOP/s; with a bias over two axes
// 475, with a cap of up to 128 450, above 730 us.  Single tokens over long caches: HBM, at the 5.2 TB/s of a
// large copy.  fp32: its matrix instructions, 127 to 133 TFLOP/s (8192 tokens, 8 heads of 64, 96 and 128) of the
// 153 of a product of 8192^3; the four-wave kernels of heads past 96 spill 46 to 75 registers.  One document of
// few row tiles leaves CUs idle: a schedule takes the place of splits of the keys, see plan().
//
// Two further forms, kernels of their own (masked_attention_window_*.hip, masked_attention_prefix_*.hip):
//
//   window      seen(i, j) and (order(j) > order(i) - window or 0 <= order(j) < sinks)
//   prefix      every key of a prefix that the batch shares, and of an entry's own keys seen(i, j)
//
// A window's waves first look over the summaries of all tiles, in parallel, and then go to those 64s of
// tiles that hold some they see; splits share out the tiles that are seen.  A mixed tile's scores are tested
// by orders, by documents where it has several, and by the end of the keys, each only where it tells: 64 keys
// 1.5 us where a whole tile takes 0.9 (all tests on each score 2.2).  8192 tokens, window of 1024, 32 heads on 8 of
// 128, bf16: 187 us, of it 8.4 for each tile of the 19 that 2048 workgroups in four rounds go over, the rest
// what each round pays to read its Q, find its tiles and write its output.  8 single tokens, 4096 of 32768
// keys: 31 us = 4.3 TB/s, and 4 for the join.  24 frames of 256 tokens, 16 heads of 64, bias over three
// axes, fp16: 78 us, the bias as above.
//
// A prefix's tiles come before an entry's own in one walk.  Where the entries have few rows each, the rows of
// all of them walk over the prefix together (it is read once, in full row tiles) and, in the same launch, each
// entry's over its own keys; a join follows.  16 x 1370 tokens after 5480, 16 heads of 64, fp16: 760 to 810 us =
// 0.76 to 0.81 PFLOP/s, as for one document of 8192.  32 single tokens after 16384 keys and over up to 700
// of their own, 32 heads on 8 of 128, bf16: 38 us = 3.3 TB/s, and 6 for the join.
//
// Both keep the probabilities of up to 32 16-bit rows of an entry in two numbers each (32 requests as above: 45 us all
// told with one number, 46 with two), and fp32 as Split has it: a tile of 32
// keys of heads of 96 takes 1150 cycles of matrix instructions (6144 of fp32 ones) and about 2700 of vector
// ones.  3 x 1500 tokens, window of 250, 8 heads on 4 of 80, cap: 60 us, by fp32 instructions 78.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.hpp"

namespace musc {
namespace mattn {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kBufferFlags = 0x00020000;   // buffer resource word 3 for raw byte-addressed loads
constexpr int kNowhere = 0x7fffff00;       // a byte offset past every extent: such loads give zeros
constexpr float kLazyLog2 = 8.f;           // the running maximum moves once a tile exceeds it by this
constexpr float kLog2e = 1.4426950408889634f;
// 16-bit types: the largest cap whose tanh is formed by one exponential and one reciprocal.  Its error,
// cap 2^-21 in the score, is then at most an eighth of what rounding a probability to fp16 (2^-11) may do.
constexpr float kSmallCap = 128.f;
constexpr int kSummaryKeys = 32;
constexpr int kMaxAxes = 3;
constexpr int kMaxSplits = 256;
constexpr int kRowTile = 128;  // rows of a workgroup of four waves
// Waves of a workgroup that share few rows' keys, for staged rows of `pitch` bytes: two tiles of 32
// keys each in 128 KiB of LDS.
constexpr int teams_of(int pitch) { return 131072 / (4 * 32 * pitch); }
constexpr int kTeamTiles = 8;  // tiles of such a wave at most
// Schedule of n row tiles, in ints: head (jobs, pieces), work (n), row tiles by their work (n), first
// job | parts << 24 of each row tile (n), jobs (row tile | part << 20 | (parts - 1) << 23), cuts (n: row |
// work before it << 7 | work from it on << 17, or 0), pieces (row tile | first row << 10 | last row << 17).
constexpr int kScheduleHead = 4, kMaxParts = 8;
__host__ __device__ inline long long schedule_jobs(long long n) { return (9 * n + 4) / 5; }
__host__ __device__ inline long long schedule_pieces(long long n) { return n + n / 4; }
__host__ __device__ inline long long schedule_block(long long n) {
  return kScheduleHead + 4 * n + schedule_jobs(n) + schedule_pieces(n);
}

template <int kDtype>
struct Type;
template <>
struct Type<MUSC_DTYPE_F32> {
  typedef float T;
  static constexpr int kTile = 32;
  static constexpr float kShift = 0.f;
};
template <>
struct Type<MUSC_DTYPE_F16> {
  typedef _Float16 T;
  typedef T Vec __attribute__((ext_vector_type(8)));
  typedef T Two __attribute__((ext_vector_type(2)));
  static constexpr int kTile = 64;
  // probabilities are formed 2^7 times as large, at most 2^15 with the slack: entries down to
  // 2^-21 of the largest stay normal fp16 numbers
  static constexpr float kShift = 7.f;
  static __device__ __forceinline__ floatx16 mfma(Vec a, Vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add_both(Two p, float sum) {
    return __builtin_amdgcn_fdot2(p, Two{(T)1.f, (T)1.f}, sum, false);
  }
};
template <>
struct Type<MUSC_DTYPE_BF16> {
  typedef __bf16 T;
  typedef T Vec __attribute__((ext_vector_type(8)));
  typedef T Two __attribute__((ext_vector_type(2)));
  static constexpr int kTile = 64;
  static constexpr float kShift = 0.f;
  static __device__ __forceinline__ floatx16 mfma(Vec a, Vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add_both(Two p, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(p, Two{(T)1.f, (T)1.f}, sum, false);
  }
};

// fp32 operands as two fp16 numbers each, x 2^n = hi + lo to 2^-22 of x, for windows and after prefixes: a
// product of two is hi hi + hi lo + lo hi, off by 3 2^-22 of itself at most, at 3/16 of the fp32 instructions'
// time.  n takes the largest of a row of Q, of a tile of K and of 32 channels of a tile's V to
// 2^13 .. 2^14, so what is below 2^-17 of that is off by 2^-39 of the largest instead.  Probabilities are
// taken 2^7 times as large, as in fp16: those below 2^-10 of a row's largest are off by 2^-32 of that.
//
// Q and K go by fp32 instructions, and Q as it is in memory, in tiles that hold infinities or NaN, or where the largest
// of a row of Q, of the tile's K and the scale are 2^kProduct and more together: below that the 2^-39 come to
// 2 D 2^(kProduct - 39) <= 2^-23 in a logit of any key, whatever the sizes of the others.
//
// Nor may V of a key that one row sees cost another its digits, so blocks of V (32 keys, 32 channels) are split if no
// entry is below 2^-kEntries of the scale, or else no key's largest entry there is below 2^-kKeys of it (of standard
// normal V one block in 20 is asked so, and none of 4000 fails).  The scale of a block stays while its largest entry is
// within 2^kFall of it; else o is taken to the block's own.
// Keys that no row of the wave sees count in none of that, whatever they hold.
//
// V's scale is 2^kMost at most and 2^-kMost of the largest entry so far at least: with probabilities up to 2^15 the
// sums over 2^31 keys stay finite, and entries from 2^-70 on stay normal numbers beside larger ones.
struct Split {
  typedef _Float16 Vec __attribute__((ext_vector_type(8)));
  static constexpr int kTop = 14, kLeast = -100, kMost = 64, kInfinity = 0x7f800000;
  static constexpr int kProduct = 8, kNever = 1000, kEntries = 17, kKeys = 6, kFall = 2;
  static constexpr float kShift = 7.f;
  static __device__ __forceinline__ floatx16 mfma(Vec a, Vec b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // e with |x| < 2^e, from the bits of |x|; the smallest share kLeast
  static __device__ __forceinline__ int exponent(int bits) { return max((bits >> 23) - 126, kLeast); }
  static __device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }
  typedef _Float16 Two __attribute__((ext_vector_type(2)));
  // two of each: hi is opaque, or the compiler forms it a second time for lo
  static __device__ __forceinline__ void split(float x, float y, float by, int j, Vec& hi, Vec& lo) {
    Two h = __builtin_convertvector((float2v{x * by, y * by}), Two);
    asm("" : "+v"(h));
    hi[j] = h[0], hi[j + 1] = h[1];
    lo[j] = (_Float16)fmaf(x, by, -(float)h[0]), lo[j + 1] = (_Float16)fmaf(y, by, -(float)h[1]);
  }
  template <typename F>
  static __device__ __forceinline__ void split(const F& a, const F& b, float by, Vec& hi, Vec& lo) {
    split(a[0], a[1], by, 0, hi, lo), split(a[2], a[3], by, 2, hi, lo);
    split(b[0], b[1], by, 4, hi, lo), split(b[2], b[3], by, 6, hi, lo);
  }
  // By its series up to 0.3 (the next term is 2^-24 of it), and 1 - 2 / (1 + e^2x): off by 2^-21 of itself, as
  // the other fp32 kernels' caps are (measured: 2^-21.8, tanhf 2^-22.6; tanhf takes 63 us where this takes 61).
  static __device__ __forceinline__ float tanh(float x) {
    const float y = x * x;
    float p = fmaf(y, 62.f / 2835.f, -17.f / 315.f);
    p = fmaf(y, p, 2.f / 15.f);
    p = fmaf(y, p, -1.f / 3.f);
    const float near = fmaf(x * y, p, x);
    const float far = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * (2.f * kLog2e))), -2.f, 1.f);
    return fabsf(x) < 0.3f ? near : far;
  }
};

// Keys of a tile: workgroups of one wave take 32, so that four of them fit a CU's LDS.
template <int kDtype, int kWaves>
constexpr int tile_keys() {
  return kWaves == 1 ? 32 : Type<kDtype>::kTile;
}

// Staged rows of K and V: 128, 256 or 512 bytes, their 16-byte chunks permuted by the row so
// that the lanes one LDS read serves together touch different banks: 16 neighbouring rows of
// one chunk (K's operands) take 16 places of a 256-byte window, and so do 4 neighbouring rows
// of 4 chunks (V's transposing reads).  Chunk c of row r is at place c ^ swizzle(r).
template <int kPitch>
__device__ __forceinline__ constexpr int swizzle(int r) {
  return kPitch == 128 ? (((r >> 1) & 1) << 2) | ((r >> 2) & 3) : ((r & 3) << 2) | ((r >> 2) & 3);
}

struct Args {
  musc_masked_attention c;
  int group, rows, row_tiles, key_tiles, splits, summaries, heads_at_once;
  int jobs;      // workgroups of a head and split: its row tiles, or the schedule's jobs
  int in_parts;  // jobs may be parts of a row tile's keys
  int in_pieces; // jobs may be the rows of a row tile before or from a document's start on
  int teams;     // waves that share few rows' keys within a workgroup
  int slots;     // workgroups that the card holds at a time
  int window, sinks;  // of windowed attention
  // prefixed attention: the prefix, its tiles (the first ones, may be none), batch entries of the grid (1 where
  // the rows of all are stacked), and whether the rows' parts are joined even if there is one
  musc_attention_prefix p;
  int p_tiles, batches, stacked, partial;
  int two_numbers;    // 16-bit types: four waves keep probabilities as two numbers
  int more_splits;    // for the join: parts over the own keys
  float *more_ml, *more_o;
  long long units;
  float* part_ml;  // (units in (b, kv head), rows, split) x (maximum, sum)
  float* part_o;   // the same x d
};

// Two calls' work in one launch.
struct TwoArgs {
  Args first, second;
  uint32_t first_blocks;
};

__device__ __forceinline__ float halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Minimum over the wave by lane-crossing moves (no LDS): lanes get their neighbours 1, 2, 4, 8 to
// the left within rows of 16, then the rows' last lanes go on to the next rows; lane 63 has it.
template <int kMove, int kRows>
__device__ __forceinline__ int min_with(int v) {
  return min(v, __builtin_amdgcn_update_dpp(0x7fffffff, v, kMove, kRows, 0xf, false));
}
__device__ __forceinline__ int wave_min_int(int v) {
  v = min_with<0x111, 0xf>(v);
  v = min_with<0x112, 0xf>(v);
  v = min_with<0x114, 0xf>(v);
  v = min_with<0x118, 0xf>(v);
  v = min_with<0x142, 0xa>(v);
  v = min_with<0x143, 0xc>(v);
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_max_int(int v) { return ~wave_min_int(~v); }
// All bits of the 32 lanes of each half, on every lane of it, in the same way.
template <int kMove, int kRows>
__device__ __forceinline__ uint32_t or_with(uint32_t v) {
  return v | (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kMove, kRows, 0xf, false);
}
__device__ __forceinline__ uint32_t halves_or(uint32_t v) {
  v = or_with<0x111, 0xf>(v);
  v = or_with<0x112, 0xf>(v);
  v = or_with<0x114, 0xf>(v);
  v = or_with<0x118, 0xf>(v);
  v = or_with<0x142, 0xa>(v);
  const uint32_t lower = __builtin_amdgcn_readlane((int)v, 31), upper = __builtin_amdgcn_readlane((int)v, 63);
  return threadIdx.x & 32 ? upper : lower;
}

// The documents and orders of a set of rows: what a tile is compared with.
struct Range {
  int dmin, dmax, omin, omax;
};

// The kernels of one storage type, each compiled in its own file (launch_all below).
void launch_f32(const Args& a, int waves, hipStream_t stream);
void launch_f16(const Args& a, int waves, hipStream_t stream);
void launch_bf16(const Args& a, int waves, hipStream_t stream);
void launch_window_f32(const Args& a, int waves, hipStream_t stream);
void launch_window_f16(const Args& a, int waves, hipStream_t stream);
void launch_window_bf16(const Args& a, int waves, hipStream_t stream);
void launch_prefix_f32(const Args& a, const Args* more, int waves, hipStream_t stream);
void launch_prefix_f16(const Args& a, const Args* more, int waves, hipStream_t stream);
void launch_prefix_bf16(const Args& a, const Args* more, int waves, hipStream_t stream);

}  // namespace mattn
}  // namespace musc
