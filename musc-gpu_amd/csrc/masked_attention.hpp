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
  long long units;
  float* part_ml;  // (units in (b, kv head), rows, split) x (maximum, sum)
  float* part_o;   // the same x d
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

// The documents and orders of a set of rows: what a tile is compared with.
struct Range {
  int dmin, dmax, omin, omax;
};

// The kernels of one storage type, each compiled in its own file (launch_all below).
void launch_f32(const Args& a, int waves, hipStream_t stream);
void launch_f16(const Args& a, int waves, hipStream_t stream);
void launch_bf16(const Args& a, int waves, hipStream_t stream);

}  // namespace mattn
}  // namespace musc
