// The attention kernel over seen keys and the join of its parts, for the files that compile
// them for one storage type each.  The mathematics is in masked_attention.hpp.
#pragma once

#include "masked_attention.hpp"

namespace musc {
namespace mattn {

template <int kN, int kI = 0, typename F>
__device__ __forceinline__ void unroll(F f) {
  if constexpr (kI < kN) {
    f(std::integral_constant<int, kI>{});
    unroll<kN, kI + 1>(f);
  }
}

// Loads straight from memory into LDS, lane l's 16 (or 4) bytes to `to` (+ kTo) + 16 l (or
// 4 l), `to` uniform.  From inline assembly, as the compiler, which cannot tell the two buffers apart,
// would wait for them before reading the other one; the loop waits for them itself.  The resource
// comes out of vector registers (v_readfirstlane), and a vector-memory instruction may read it from the
// fifth wait state after that on, which the compiler does not see to for an asm statement: the scalar
// instruction and s_nop 3 are five.  (M0 needs one.)
template <int kTo>
__device__ __forceinline__ void load_to_lds_16(uint32_t to, int offset, int4v from, int from_offset) {
  asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(to), "v"(offset), "s"(from), "s"(from_offset), "i"(kTo) : "memory", "m0", "scc");
}
__device__ __forceinline__ void load_to_lds_4(const void* place, int offset, int4v from) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(lds_void*)place);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(to), "v"(offset), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ int4v resource(const void* base, long long bytes) {
  const unsigned long long at = reinterpret_cast<unsigned long long>(base);
  return int4v{__builtin_amdgcn_readfirstlane((int)(uint32_t)at), __builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)),
               __builtin_amdgcn_readfirstlane((int)bytes), kBufferFlags};
}

// kWaves waves of 32 rows each; kD: head width rounded up to 64, 96 or 128; kMode: kCapped,
// kBiased and, with four waves, kInParts in any combination (without them their tests and registers
// are not in the key loop: 155 -> 127 us for 256 workgroups of 128 tiles, one per CU, fp16, kD = 64;
// kInParts alone costs 3 to 8 %).  kTeams > 1 (with one wave): that many waves take every n-th tile of
// the same rows, each with its own place in LDS and at its own pace, and join their parts there.
// kEither: a cap and a bias if the call has them, tested per tile (for the kernels of few rows and
// of parts, which wait for memory or for one another).  kLargeCap (16-bit types, with kEither): the cap is past
// kSmallCap; kernels of their own, as tanhf beside the other form costs registers (parts of fp16 heads of 64:
// 76 spilled instead of 17): 8192 tokens, 16 heads of 64, fp16, 730 us past kSmallCap, 450 up to it.
// kWindowed: keys behind the window and past the sinks are not seen either.  kPrefixed: the first a.p_tiles
// tiles are of a prefix that the batch shares; a.stacked: all rows of the batch over those tiles.  kTwoNumbers (16-bit
// types, four waves): probabilities as two numbers, as single waves have them.
constexpr int kCapped = 1, kBiased = 2, kInParts = 4, kEither = 8, kLargeCap = 16, kWindowed = 32, kPrefixed = 64,
              kTwoNumbers = 128;
template <int kDtype, int kD, int kWaves, int kTeams, int kMode>
__device__ __forceinline__ void attention_of_block(const Args& a, const uint32_t block, const uint32_t blocks) {
  using Ty = Type<kDtype>;
  typedef typename Ty::T T;
  constexpr bool k16 = kDtype != MUSC_DTYPE_F32;
  constexpr int kTile = tile_keys<kDtype, kWaves>(), kSub = kTile / 32;
  constexpr int kPer = 16 / (int)sizeof(T);                 // elements of a 16-byte chunk
  constexpr int kPitch = (kD <= 64 ? 64 : 128) * (int)sizeof(T);
  constexpr int kPlaces = kPitch / 16;                      // chunks of a staged row
  constexpr int kPart = kTile * kPitch;                     // bytes of a staged K or V tile
  constexpr int kLoads = kPart / 1024 / kWaves;             // loads of K (and of V) per wave
  static_assert(kLoads * kWaves * 1024 == kPart, "whole loads per wave");
  constexpr int kO = kD / 32;
  constexpr bool windowed = (kMode & kWindowed) != 0, prefixed = (kMode & kPrefixed) != 0;
  // fp32 as three fp16 products, see Split in masked_attention.hpp
  constexpr bool kSplit = !k16 && (windowed || prefixed);
  constexpr float kShift = kSplit ? Split::kShift : Ty::kShift;
  // few 16-bit rows of windows and prefixes: probabilities as two numbers each.  Their second product is in the
  // shadow of the loads, and with rounded ones a few rows may be twice as far from float64 as their own rounding
  // leaves them; over many rows it is 1.2 to 1.3 times (and two numbers 10 to 39 % of the time).  Few rows of each of many entries likewise, so that an
  // entry's output does not hang on how many others share its call.
  constexpr bool kTwoTerms = k16 && (windowed || prefixed) && (kWaves == 1 || (kMode & kTwoNumbers) != 0);
  __shared__ __attribute__((aligned(1024))) char staged[2 * kTeams][2 * kPart];
  __shared__ __attribute__((aligned(16))) int docs_s[2 * kTeams][64], ords_s[2 * kTeams][64];
  __shared__ float pos_s[2 * kTeams][64 * kMaxAxes];
  __shared__ Range ranges[kWaves];
  __shared__ unsigned long long chunks_s[windowed ? kWaves * kTeams : 1];
  __shared__ int seen_s[windowed ? kWaves * kTeams : 1];

  const musc_masked_attention& c = a.c;
  // uniform numbers in scalar registers (the divisions leave them in vector ones)
  const auto uniform = [](long long x) { return __builtin_amdgcn_readfirstlane((int)x); };
  uint32_t split, job, bh;
  if (a.heads_at_once) {
    // one XCD works on heads_at_once heads together, row tile by row tile (the longest first)
    const uint32_t per_xcd = (uint32_t)((prefixed ? a.batches : c.batch) * c.kv_heads) / kXcds, local = block / kXcds;
    const uint32_t of_group = (uint32_t)(a.heads_at_once * a.jobs * a.splits);
    const uint32_t group = uniform(local / of_group), in_group = local - group * of_group;
    const uint32_t first = group * a.heads_at_once, at_once = min((uint32_t)a.heads_at_once, per_xcd - first);
    const uint32_t rest = uniform(in_group / a.splits);
    split = in_group - rest * a.splits;
    job = uniform(rest / at_once);
    bh = block % kXcds * per_xcd + first + (rest - job * at_once);
  } else {
    const uint32_t unit = (block % kXcds) * (blocks / kXcds) + block / kXcds;
    if (unit >= (uint32_t)a.units) return;
    const uint32_t rest = uniform(unit / a.splits);
    split = unit - rest * a.splits;
    bh = uniform(rest / a.jobs);
    job = rest - bh * a.jobs;
  }
  // a shared prefix's heads are neighbours over the batch, so that an XCD reads it once for many of them
  const int of_major = prefixed ? a.batches : c.kv_heads, major = uniform(bh / of_major), minor = bh - major * of_major;
  const int b = prefixed ? minor : major, kvh = prefixed ? major : minor;
  const int tid = threadIdx.x, lane = tid % kWave;
  const int team = kTeams > 1 ? __builtin_amdgcn_readfirstlane(tid / kWave) : 0;
  const int wave = kTeams > 1 ? 0 : __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lq = lane & 31, lh = lane >> 5;

  // tiles of this split (of a window: all of them, and every splits-th of those that are seen), 64 sorted
  // at a time by the keys' summary; the first 64 are asked for now
  const int lo = windowed ? 0 : uniform((long long)a.key_tiles * split / a.splits);
  const int hi = windowed ? a.key_tiles : uniform((long long)a.key_tiles * (split + 1) / a.splits);
  const int p_tiles = prefixed ? a.p_tiles : 0;
  const int4* summary = c.k_summary ? reinterpret_cast<const int4*>(c.k_summary) + b * c.k_summary_sb : nullptr;
  auto summary_of = [&](int t) __attribute__((always_inline)) {
    int4 k = make_int4(0, 0, 0, 0);
    if (summary && t >= (prefixed ? max(lo, p_tiles) : lo) && t < hi) {
      t -= p_tiles;
      k = summary[(long long)t * kSub];
      if (kSub > 1 && t * kSub + 1 < a.summaries) {
        const int4 n = summary[(long long)t * kSub + 1];
        k = make_int4(min(k.x, n.x), max(k.y, n.y), min(k.z, n.z), max(k.w, n.w));
      }
    }
    return k;
  };
  const int4 first_summary = summary_of(lo / 64 * 64 + lane);
  // a window's tiles are all looked at before the first: each wave takes every n-th 64, the first ones
  // asked for now too
  constexpr int kAll = kWaves * kTeams, kAhead = !windowed ? 0 : kAll == 1 ? 16 : 4;
  const int self = windowed ? __builtin_amdgcn_readfirstlane(tid / kWave) : 0;
  const bool look = windowed && (hi > 64 || (kTeams == 1 && a.splits > 1));
  int4 ahead[windowed ? kAhead : 1];
  if (look) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = summary_of((self + i * kAll) * 64 + lane);
  }

  // the row tile, or the part of its keys, that the schedule names; without one later rows first:
  // with an order of tokens they see more keys, and the longest work should not start last
  constexpr bool in_parts = (kMode & kInParts) != 0;
  int tile_of_rows = a.row_tiles - 1 - (int)job, part = team, parts = kTeams;
  if (windowed && kTeams == 1) part = (int)split, parts = a.splits;
  int first_row = 0, last_row = kRowTile - 1;
  if (kWaves > 1 && c.schedule) {
    const int* schedule = c.schedule + b * c.schedule_sb;
    if constexpr (in_parts) {
      const int jobs = schedule[0], j = schedule[kScheduleHead + 3 * a.row_tiles + job];
      if ((int)job >= jobs) return;
      tile_of_rows = uniform(j & 0xfffff);
      part = uniform((j >> 20) & 7);
      parts = uniform(((j >> 23) & 7) + 1);
    } else {
      const int pieces = schedule[1];
      const int e = schedule[kScheduleHead + job + (a.in_pieces ? 4 * a.row_tiles + (int)schedule_jobs(a.row_tiles) : a.row_tiles)];
      if (a.in_pieces) {
        if ((int)job >= pieces) return;
        first_row = uniform((e >> 10) & 127), last_row = uniform((e >> 17) & 127);
      }
      tile_of_rows = uniform(e & 1023);
    }
  }
  tile_of_rows = min(max(tile_of_rows, 0), a.row_tiles - 1);
  const int row = (tile_of_rows * kWaves + wave) * 32 + lq;
  const bool inside = row < a.rows && (in_parts || kWaves == 1 || (wave * 32 + lq >= first_row && wave * 32 + lq <= last_row));
  int token = inside ? (int)((uint32_t)row / (uint32_t)a.group) : 0;
  const int head = kvh * a.group + (inside ? row - token * a.group : 0);
  int qb = b;  // the batch entry of this row
  if (prefixed && a.stacked) {
    qb = (int)((uint32_t)token / (uint32_t)c.q_len);
    token -= qb * c.q_len;
  }
  const int d = c.d, k_len = c.k_len, axes = kMode & (kBiased | kEither) ? c.axes : 0;

  // this row's document and order (rows outside the tensor read token 0's), its Q and positions,
  // all asked for before any is used
  int qdoc = 0, qord = 0;
  if (c.q_documents) qdoc = c.q_documents[qb * c.q_tokens_sb + token];
  if (c.q_order) qord = c.q_order[qb * c.q_tokens_sb + token];
  const T* qrow = static_cast<const T*>(c.q) + qb * c.q_sb + (long long)token * c.q_st + head * c.q_sh;
  constexpr int kQ = kD / (2 * kPer);
  typedef T TVec __attribute__((ext_vector_type(kPer)));
  TVec qf[kQ];
#pragma unroll
  for (int m = 0; m < kQ; ++m) {
    const int at = (2 * m + lh) * kPer;
    qf[m] = TVec{};
    if (at < d) qf[m] = *reinterpret_cast<const TVec*>(qrow + at);
  }
  float qpos[kMaxAxes], slope[kMaxAxes];
#pragma unroll
  for (int x = 0; x < kMaxAxes; ++x) {
    qpos[x] = 0.f, slope[x] = 0.f;
    if (x < axes) {
      qpos[x] = c.q_positions[qb * c.q_positions_sb + (long long)token * axes + x];
      slope[x] = c.slopes[head * axes + x];
    }
  }

  const bool live = inside && qdoc >= 0;
  Range mine, all_rows;
  mine.dmin = wave_min_int(live ? qdoc : 0x7fffffff);
  mine.dmax = wave_max_int(live ? qdoc : -1);
  mine.omin = wave_min_int(live ? qord : 0x7fffffff);
  mine.omax = wave_max_int(live ? qord : (int)0x80000000);
  all_rows = mine;
  if constexpr (kWaves > 1) {
    if (lane == 0) ranges[wave] = mine;
  }
  // keys of calls without documents or orders have 0
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) docs_s[2 * team + i][lane] = 0, ords_s[2 * team + i][lane] = 0;
  }
  __syncthreads();
  if constexpr (kWaves > 1) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      all_rows.dmin = min(all_rows.dmin, ranges[w].dmin);
      all_rows.dmax = max(all_rows.dmax, ranges[w].dmax);
      all_rows.omin = min(all_rows.omin, ranges[w].omin);
      all_rows.omax = max(all_rows.omax, ranges[w].omax);
    }
  }

  // Of a window: the order of the first key in it, and which 64s of tiles hold some that the workgroup's rows
  // see (bit 63: all from the 63rd on), found by all waves before any of them has its accumulators; and of
  // the splits only as many as there are such tiles (four of them for four waves) have work.
  const auto window_from = [&](int order) { return __builtin_elementwise_sub_sat(order, a.window - 1); };
  auto may_see_tile = [&](const int4 k, const Range& r) __attribute__((always_inline)) {  // without branches
    bool may = (k.y >= 0) & (k.x <= r.dmax) & (k.y >= r.dmin) & (k.z <= r.omax);
    if (windowed) may &= (k.w >= window_from(r.omin)) | ((k.w >= 0) & (k.z < a.sinks));
    return may;
  };
  unsigned long long chunks = ~0ull;
  constexpr int kLeast = kDtype == MUSC_DTYPE_F32 ? 2 : 4;  // tiles of a split
  if constexpr (windowed) {
    if (look) {
      unsigned long long here = 0;
      int seen_tiles = 0;
      auto look_at = [&](int n, const int4 k) __attribute__((always_inline)) {
        const unsigned long long some = __ballot(n * 64 + lane < hi && may_see_tile(k, all_rows));
        if (some) here |= 1ull << min(n, 63);
        seen_tiles += __popcll(some);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) look_at(self + i * kAll, ahead[i]);
#pragma unroll 4
      for (int n = self + kAhead * kAll; n * 64 < hi; n += kAll) look_at(n, summary_of(n * 64 + lane));
      if (lane == 0) chunks_s[self] = here, seen_s[self] = seen_tiles;
      __syncthreads();
      chunks = 0, seen_tiles = 0;
#pragma unroll
      for (int w = 0; w < kAll; ++w) chunks |= chunks_s[w], seen_tiles += seen_s[w];
      chunks = (unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(chunks >> 32)) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((int)chunks);
      if (kTeams == 1 && a.splits > 1) {
        seen_tiles = __builtin_amdgcn_readfirstlane(seen_tiles);
        parts = max(min(parts, kWaves == 1 ? seen_tiles : (seen_tiles + kLeast - 1) / kLeast), 1);
        if (part >= parts) {  // the whole workgroup
          if (inside && lh == 0)
            reinterpret_cast<float2*>(a.part_ml)[((long long)bh * a.rows + row) * a.splits + split] = make_float2(-INFINITY, 0.f);
          return;
        }
      }
    }
  }

  // Scores stay "raw" until the exponential: score in log2 units =
  // raw * to_log2 (+ a constant that cancels), to_log2 > 0:
  //   no cap   raw = +- q . k (Q negated for a negative scale), to_log2 = |scale| log2 e
  //   cap      raw = -1 / (1 + e^2x), x = scale q . k / cap, as cap tanh x = cap (1 + 2 raw): off by
  //            cap 2^-21 however small the score is, so in 16-bit types up to kSmallCap only;
  //            raw = tanh x above it and in fp32, off by the score's own 2^-21
  const bool capped = (kMode & kCapped) != 0 || ((kMode & kEither) != 0 && c.cap > 0.f);
  constexpr bool by_exponential = k16 && (kMode & kLargeCap) == 0;
  const float scale = c.scale == 0.f ? 1.f : c.scale;
  const float to_log2 = (capped ? (by_exponential ? 2.f * c.cap : c.cap) : fabsf(scale)) * kLog2e;
  const float by_cap = capped ? scale / c.cap * (by_exponential ? 2.f * kLog2e : 1.f) : 0.f;
  const bool negate = !capped && scale < 0.f;
#pragma unroll
  for (int m = 0; m < kQ; ++m) {
    if (negate) qf[m] = -qf[m];
    if (c.scale == 0.f) qf[m] = TVec{};
  }
  // split: this row's Q in 2^(q_exp - 14), and the K (k_exp) up to which the wave's rows bear splitting
  Split::Vec qh[kSplit ? kQ / 2 : 1], ql[kSplit ? kQ / 2 : 1];
  int q_exp = 0, k_most = 0;
  if constexpr (kSplit) {
    float most = 0.f;
#pragma unroll
    for (int m = 0; m < kQ; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) most = __builtin_elementwise_maximum(most, fabsf(qf[m][j]));
    most = halves_max(most);
    q_exp = Split::exponent(__float_as_int(most));
    k_most = Split::kProduct - Split::exponent(__float_as_int(fabsf(scale))) -
             wave_max_int(!live ? Split::kLeast : most < INFINITY ? q_exp : Split::kNever);
    const float by = Split::power(Split::kTop - q_exp);
#pragma unroll
    for (int m = 0; m < kQ; m += 2) Split::split(qf[m], qf[m + 1], by, qh[m / 2], ql[m / 2]);
  }
  // the B operand of the distances: 1 and -position; slopes in raw units
#pragma unroll
  for (int x = 0; x < kMaxAxes; ++x) {
    qpos[x] = x < axes ? (lh == 0 ? 1.f : -qpos[x]) : 0.f;
    slope[x] = slope[x] * kLog2e / to_log2;
  }

  // Staging: load i of a tile fills 1024 bytes, whole rows; wave w issues loads w, w + kWaves, ..
  // The loads of a whole tile share a resource based at the wave's first row, and a scalar offset
  // leads to the rows of each; in the last, partial tile each has a resource of its own that ends
  // with the last key.  Lanes of channels past d load from nowhere.
  const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(c.k) + b * c.k_sb + (long long)kvh * c.k_sh);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(c.v) + b * c.v_sb + (long long)kvh * c.v_sh);
  const uint32_t own_k_row = (uint32_t)(c.k_st * (long long)sizeof(T)), own_v_row = (uint32_t)(c.v_st * (long long)sizeof(T));
  const char *pkbase = kbase, *pvbase = vbase;
  uint32_t p_k_row = 0, p_v_row = 0;
  if constexpr (prefixed) {
    pkbase = reinterpret_cast<const char*>(static_cast<const T*>(a.p.k) + (long long)kvh * a.p.k_sh);
    pvbase = reinterpret_cast<const char*>(static_cast<const T*>(a.p.v) + (long long)kvh * a.p.v_sh);
    p_k_row = (uint32_t)(a.p.k_st * (long long)sizeof(T)), p_v_row = (uint32_t)(a.p.v_st * (long long)sizeof(T));
  }
  const uint32_t staged_at = (uint32_t)(size_t)(lds_void*)&staged[0][0] + wave * 1024;
  constexpr int kRows = 64 / kPlaces;  // rows of a load
  const int row_bytes = d * (int)sizeof(T);
  auto load_tile = [&](int tile, int buf) __attribute__((always_inline)) {
    const bool shared = prefixed && tile < p_tiles;
    const int first = (shared ? tile : tile - p_tiles) * kTile, mine = wave * kRows;
    const int rem = min((shared ? a.p.len : k_len) - first, kTile);
    const uint32_t k_row = shared ? p_k_row : own_k_row, v_row = shared ? p_v_row : own_v_row;
    const uint32_t to = __builtin_amdgcn_readfirstlane(staged_at + buf * 2 * kPart);
    const char* kt = (shared ? pkbase : kbase) + (unsigned long long)(uint32_t)(first + mine) * k_row;
    const char* vt = (shared ? pvbase : vbase) + (unsigned long long)(uint32_t)(first + mine) * v_row;
    auto lane_offset = [&](int j, uint32_t row) {
      const int r = lane / kPlaces, chunk = (lane % kPlaces) ^ swizzle<kPitch>((wave + kWaves * j) * kRows + r);
      return chunk * kPer < d ? (int)(r * row) + chunk * 16 : kNowhere;
    };
    if (rem == kTile) {
      const int4v rk = resource(kt, (long long)(kTile - mine - 1) * k_row + row_bytes);
      const int4v rv = resource(vt, (long long)(kTile - mine - 1) * v_row + row_bytes);
      unroll<kLoads>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        load_to_lds_16<j * kWaves * 1024>(to, lane_offset(j, k_row), rk, (int)(j * kWaves * kRows * k_row));
        load_to_lds_16<j * kWaves * 1024 + kPart>(to, lane_offset(j, v_row), rv, (int)(j * kWaves * kRows * v_row));
      });
    } else {
      unroll<kLoads>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int rows = rem - mine - j * kWaves * kRows;
        const unsigned long long at = j * kWaves * kRows;
        load_to_lds_16<j * kWaves * 1024>(
            to, lane_offset(j, k_row), resource(kt + at * k_row, rows > 0 ? (long long)(rows - 1) * k_row + row_bytes : 0), 0);
        load_to_lds_16<j * kWaves * 1024 + kPart>(
            to, lane_offset(j, v_row), resource(vt + at * v_row, rows > 0 ? (long long)(rows - 1) * v_row + row_bytes : 0), 0);
      });
    }
    if (wave == kWaves - 1) {
      if (c.k_documents && !shared)
        load_to_lds_4(&docs_s[buf][0], lane * 4,
                      resource(c.k_documents + b * c.k_tokens_sb + first, rem * 4));
      if (c.k_order && !shared)
        load_to_lds_4(&ords_s[buf][0], lane * 4,
                      resource(c.k_order + b * c.k_tokens_sb + first, rem * 4));
      if (axes) {
        const float* positions = shared ? a.p.positions : c.k_positions + b * c.k_positions_sb;
        const int4v rp = resource(positions + (long long)first * axes, rem * axes * 4);
#pragma unroll
        for (int x = 0; x < kMaxAxes; ++x)
          if (x < axes) load_to_lds_4(&pos_s[buf][64 * x], (64 * x + lane) * 4, rp);
      }
    }
  };

  floatx16 o[kO];
  int v_exp[kSplit ? kO : 1], v_top[kSplit ? kO : 1];  // split: o is in 2^(v_exp - 14); the largest entry so far
  float m_run, l_run;  // running maximum (raw) and sum of this half's keys
  float base;          // exponent of a score: raw * to_log2 + base
  bool mixed_seen;

  // one staged tile; whole: every row sees every key.  careful: in a mixed tile, products
  // of keys that a row does not see are left out one by one (their V may be infinite or NaN)
  auto attend = [&](int buf, int tile, bool whole, bool one, auto careful_c, auto read) __attribute__((always_inline)) {
    constexpr bool careful = decltype(careful_c)::value;
    // Byte places of this lane's operands: row lq (K) or the row and chunk of its V operand, in
    // chunk order from the permutation's exclusive or, which all further chunks keep.  Formed
    // anew for each tile, as keeping all of them would take the registers of the operands.
    int k_at = buf * 2 * kPart + lq * kPitch + ((lh ^ swizzle<kPitch>(lq)) << 4);
    int v_at = buf * 2 * kPart + kPart;
    if constexpr (k16) {
      const int r = 4 * lh + ((lq & 15) >> 2);
      v_at += r * kPitch + (((2 * (lq >> 4) + ((lq & 3) >> 1)) ^ swizzle<kPitch>(r)) << 4) + 8 * (lq & 1);
    } else {
      v_at += 4 * lh * kPitch + (((lq >> 2) ^ lh) << 4) + 4 * (lq & 3);
    }
    asm volatile("" : "+v"(k_at), "+v"(v_at));
    const char* all = &staged[0][0];
    floatx16 s[kSub];
    TVec kf[kSub][kQ];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int m = 0; m < kQ; ++m)
        kf[u][m] = *reinterpret_cast<const TVec*>(all + (k_at ^ (m << 5)) + 32 * u * kPitch);
    __builtin_amdgcn_sched_barrier(0);  // all reads in flight before the first product waits
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = 0.f;
    if constexpr (kSplit) {
      float most = 0.f;
#pragma unroll
      for (int m = 0; m < kQ; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) most = __builtin_elementwise_maximum(most, fabsf(kf[0][m][j]));
      // this lane's key's largest entry; one that no row of the wave sees does not count
      bool counts = true;
      if (!whole && !(prefixed && tile < p_tiles)) {
        const int kd = docs_s[buf][lq], ko = ords_s[buf][lq];
        counts = (kd >= mine.dmin) & (kd <= mine.dmax) & (ko <= mine.omax);
        if (windowed) counts &= (ko >= window_from(mine.omin)) | ((uint32_t)ko < (uint32_t)a.sinks);
      }
      const int largest = wave_max_int(counts ? __float_as_int(most) : 0), k_exp = Split::exponent(largest);
      int by = 0;  // exponent of the products
      if (!careful && largest < Split::kInfinity && k_exp <= k_most) {
        const float k_by = Split::power(Split::kTop - k_exp);
        by = k_exp + q_exp - 2 * Split::kTop;
#pragma unroll
        for (int m = 0; m < kQ / 2; ++m) {
          Split::Vec kh, kl;
          Split::split(kf[0][2 * m], kf[0][2 * m + 1], k_by, kh, kl);
          s[0] = Split::mfma(kl, qh[m], s[0]);
          s[0] = Split::mfma(kh, ql[m], s[0]);
          s[0] = Split::mfma(kh, qh[m], s[0]);
          __builtin_amdgcn_sched_barrier(0);  // one pair's registers at a time
        }
      } else {
        // Q as it is, read again: its parts have 22 bits only
        int from = token;
        asm volatile("" : "+v"(from));  // its address is formed here, not kept beside the parts
        const T* again = static_cast<const T*>(c.q) + qb * c.q_sb + (long long)from * c.q_st + head * c.q_sh;
#pragma unroll
        for (int m = 0; m < kQ; ++m) {
          const int at = (2 * m + lh) * kPer;
          TVec q = TVec{};
          if (at < d && c.scale != 0.f) q = *reinterpret_cast<const TVec*>(again + at);
          if (negate) q = -q;
#pragma unroll
          for (int j = 0; j < 4; ++j) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[0][m][j], q[j], s[0], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) s[0][v] = __builtin_ldexpf(s[0][v], by);
    } else {
#pragma unroll
    for (int m = 0; m < kQ; ++m)
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        if constexpr (k16) {
          s[u] = Ty::mfma(kf[u][m], qf[m], s[u]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[u][m][j], qf[m][j], s[u], 0, 0, 0);
        }
      }
    }
    // V^T fragments by transposing LDS reads, in flight during the softmax: within a group of 16
    // lanes, lane i's element j is element i % 4 of the 8 bytes that lane 4 j + i / 4 addressed,
    // so with V row-major the lane that addresses V[key0 + r / 4][d0 + 4 (r % 4) ..] (r its place
    // in the group) hands element j of lane i the value V[key0 + j][d0 + i]: the A operand's row
    // d0 + i, k = j
    short8v vf[k16 && !careful ? 2 * kSub : 1][k16 && !careful ? kO : 1];
    auto read_v = [&](int mm, int x) {
      // key0 = 16 mm + 4 lh (+ 8: the permutation's bit 1), d0 = 32 x + 16 (lq / 16)
      auto tr = [&](int upper) {
        typedef __attribute__((address_space(3))) short4v lds_short4v;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_short4v*)(all + (v_at ^ (x << 6) ^ (upper << 5)) + (16 * mm + 8 * upper) * kPitch));
      };
      const short4v f0 = tr(0), f1 = tr(1);
      return short8v{f0[0], f0[1], f0[2], f0[3], f1[0], f1[1], f1[2], f1[3]};
    };
    if constexpr (k16 && !careful) {
#pragma unroll
      for (int mm = 0; mm < 2 * kSub; ++mm)
#pragma unroll
        for (int x = 0; x < kO; ++x) vf[mm][x] = read_v(mm, x);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (capped) {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float x = s[u][v] * by_cap;
          s[u][v] = by_exponential ? __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x)) : kSplit ? Split::tanh(x) : tanhf(x);
        }
    }
    // distances from the matrix cores: position(j) * 1 + 1 * -position(i), exact in fp32
#pragma unroll
    for (int x = 0; x < kMaxAxes; ++x)
      if (x < axes)
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          floatx16 apart;
#pragma unroll
          for (int v = 0; v < 16; ++v) apart[v] = 0.f;
          const float kp = pos_s[buf][(32 * u + lq) * axes + x];
          apart = __builtin_amdgcn_mfma_f32_32x32x2f32(lh == 0 ? kp : 1.f, qpos[x], apart, 0, 0, 0);
#pragma unroll
          for (int v = 0; v < 16; ++v) s[u][v] = fmaf(-slope[x], fabsf(apart[v]), s[u][v]);
        }
    // register v of block u holds key 32 u + 8 (v / 4) + 4 lh + v % 4
    uint32_t seen = 0xffffffffu;
    if (!whole) {
      mixed_seen = true;
      // this row's window: its first order and how many follow, and its sinks; formed anew, as v_at is
      int order = qord;
      if (windowed) asm volatile("" : "+v"(order));
      const int qfirst = windowed ? window_from(order) : 0;
      const uint32_t qspan = (uint32_t)order - (uint32_t)qfirst;
      const uint32_t qsinks = windowed && order >= 0 && a.sinks > 0 ? (uint32_t)min(order, a.sinks - 1) + 1 : 0;
      const bool shared = prefixed && tile < p_tiles;
      const int rem = shared ? a.p.len - tile * kTile : k_len - (tile - p_tiles) * kTile;
      if constexpr (windowed || prefixed) {
        // orders, documents where the tile has more than one, and the end of the keys, one after the other
        auto only = [&](auto seen_if) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool see = seen_if(32 * u + 8 * g + 4 * lh, i);
                s[u][4 * g + i] = see ? s[u][4 * g + i] : -INFINITY;
                if (careful && !see) seen &= ~(1u << (16 * u + 4 * g + i));
              }
        };
        if (!shared) {
          only([&](int key, int i) __attribute__((always_inline)) {
            const int ko = ords_s[buf][key + i];
            return windowed ? ((uint32_t)ko - (uint32_t)qfirst <= qspan) | ((uint32_t)ko < qsinks) : ko <= order;
          });
          if (!one)
            only([&](int key, int i) __attribute__((always_inline)) { return docs_s[buf][key + i] == qdoc; });
        }
        if (rem < kTile) only([&](int key, int i) __attribute__((always_inline)) { return key + i < rem; });
      } else
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int key = 32 * u + 8 * g + 4 * lh;
          const int4v kd = *reinterpret_cast<const int4v*>(&docs_s[buf][key]);
          const int4v ko = *reinterpret_cast<const int4v*>(&ords_s[buf][key]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool see = kd[i] == qdoc && ko[i] <= qord && key + i < rem;
            s[u][4 * g + i] = see ? s[u][4 * g + i] : -INFINITY;
            if (careful && !see) seen &= ~(1u << (16 * u + 4 * g + i));
          }
        }
    }
    if constexpr (!careful) read();  // the tile's LDS is not read any more, in 16-bit types
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) top = __builtin_elementwise_maximum(top, s[u][v]);
    top = halves_max(top);
    if (!__all((top - m_run) * to_log2 <= kLazyLog2)) {  // false at first, and for NaN
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * to_log2);
      l_run *= alpha;
#pragma unroll
      for (int x = 0; x < kO; ++x)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[x][v] *= alpha;
      m_run = m_new;
      base = kShift - (m_run == -INFINITY ? 0.f : m_run * to_log2);
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = __builtin_amdgcn_exp2f(fmaf(s[u][v], to_log2, base));
    TVec p[2 * kSub], rest[kTwoTerms ? 2 * kSub : 1];
    if constexpr (kTwoTerms) {
#pragma unroll
      for (int mm = 0; mm < 2 * kSub; ++mm)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f = s[mm >> 1][8 * (mm & 1) + j];
          p[mm][j] = (T)f;
          rest[mm][j] = (T)(f - (float)p[mm][j]);
          l_run += f;
        }
    } else if constexpr (k16) {
#pragma unroll
      for (int mm = 0; mm < 2 * kSub; ++mm)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float2v f = {s[mm >> 1][8 * (mm & 1) + j], s[mm >> 1][8 * (mm & 1) + j + 1]};
          const auto two = __builtin_convertvector(f, typename Ty::Two);
          p[mm][j] = two[0], p[mm][j + 1] = two[1];
          l_run = Ty::add_both(two, l_run);  // the sum of what the product uses
        }
    } else {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) l_run += s[u][v];
    }
    if (careful && !whole) {
#pragma unroll 1
      for (int key = 0; key < kTile; ++key) {
        const int u0 = key >> 5, v0 = ((key & 31) >> 3) * 4 + (key & 3), from = lq + 32 * ((key >> 2) & 1);
        float pr = 0.f;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (u == u0 && v == v0) pr = kTwoTerms ? s[u][v] : (float)(T)s[u][v];
        pr = __shfl(pr, from, kWave);
        const bool see = (__shfl(seen, from, kWave) >> (16 * u0 + v0)) & 1;
#pragma unroll
        for (int x = 0; x < kO; ++x)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            if (v % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // few values at a time
            const int at = 32 * x + 8 * (v >> 2) + 4 * lh + (v & 3);
            const T value = *reinterpret_cast<const T*>(staged[buf] + kPart + key * kPitch + ((at / kPer) ^ swizzle<kPitch>(key)) * 16 +
                                                        at % kPer * (int)sizeof(T));
            if (see) o[x][v] = fmaf(pr, (float)value, o[x][v]);
          }
      }
      return;
    }
    if constexpr (k16) {
#pragma unroll
      for (int mm = 0; mm < 2 * kSub; ++mm)
#pragma unroll
        for (int x = 0; x < kO; ++x) {
          const TVec values = __builtin_bit_cast(TVec, careful ? read_v(mm, x) : vf[careful ? 0 : mm][careful ? 0 : x]);
          if constexpr (kTwoTerms) o[x] = Ty::mfma(values, rest[mm], o[x]);
          o[x] = Ty::mfma(values, p[mm], o[x]);
        }
    } else if constexpr (kSplit) {
      Split::Vec ph[2], pl[2];
      auto scale_to = [&](int x, int to) __attribute__((always_inline)) {
#pragma unroll
        for (int v = 0; v < 16; ++v) o[x][v] = __builtin_ldexpf(o[x][v], v_exp[x] - to);
        v_exp[x] = to;
      };
      uint32_t used = 0xffffu;  // of this half's keys, those (by element) that some row sees
      if (!careful && !whole) {
        used = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) used |= min(__float_as_uint(s[0][e]), 1u) << e;
        used = halves_or(live ? used : 0);
      }
      // The smallest of the used keys (lane lq has key lq) by their largest entries of block x; zeros do not count.
      auto smallest_key = [&](int x) __attribute__((always_inline)) {
        float most = 0.f;
#pragma unroll
        for (int m = 4 * x; m < 4 * x + 4; ++m) {
          const TVec row = *reinterpret_cast<const TVec*>(all + ((k_at + kPart) ^ (m << 5)));
#pragma unroll
          for (int j = 0; j < 4; ++j) most = __builtin_elementwise_maximum(most, fabsf(row[j]));
        }
        most = halves_max(most);
        const uint32_t used_there = (uint32_t)__shfl((int)used, 32 * ((lq >> 2) & 1), kWave);
        const bool counts = ((used_there >> ((lq >> 3) * 4 + (lq & 3))) & 1) & (most != 0.f);
        return __int_as_float(wave_min_int(counts ? __float_as_int(most) : Split::kInfinity));
      };
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int j = 0; j < 8; j += 2) Split::split(s[0][8 * g + j], s[0][8 * g + j + 1], 1.f, j, ph[g], pl[g]);
#pragma unroll
      for (int x = 0; x < kO; ++x) {
        float f[16];  // element e: key 8 (e / 4) + 4 lh + e % 4, channel 32 x + lq
        float most = 0.f, least = INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f[e] = *reinterpret_cast<const float*>(
              all + (v_at ^ (x << 7) ^ ((e & 3) << 6) ^ (((e >> 2) & 1) << 5)) + (8 * (e >> 2) + (e & 3)) * kPitch);
          if (!careful) {
            const int bits = __float_as_int(f[e]), mask = __builtin_amdgcn_sbfe((int)used, e, 1);
            least = __builtin_elementwise_minimum(least, fabsf(__int_as_float((bits & mask) | (Split::kInfinity & ~mask))));
            f[e] = __int_as_float(bits & mask);
          }
          most = __builtin_elementwise_maximum(most, fabsf(f[e]));
        }
        // The block's scale: as it was, or, where its largest entry has left that, its own; and whether it fits
        // all entries, or all keys by their largest.
        const int bits = wave_max_int(__float_as_int(most)), here = Split::exponent(bits);
        const bool kept = bits == 0 || (here <= v_exp[x] && here >= v_exp[x] - Split::kFall);
        const int to = kept ? v_exp[x] : max(here, v_top[x] - Split::kMost);
        bool fits = !careful && bits < Split::kInfinity && to <= Split::kMost;
        if (fits && __any((32 * x + lq < d) & (least < Split::power(to - Split::kEntries))))
          fits = smallest_key(x) >= Split::power(to - Split::kKeys);
        if (fits) {
          if (to != v_exp[x]) scale_to(x, to);
          v_top[x] = max(v_top[x], to);
          const float by = Split::power(Split::kTop - to);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            Split::Vec vh, vl;
            Split::split(float4{f[8 * g], f[8 * g + 1], f[8 * g + 2], f[8 * g + 3]},
                         float4{f[8 * g + 4], f[8 * g + 5], f[8 * g + 6], f[8 * g + 7]}, by, vh, vl);
            o[x] = Split::mfma(vl, ph[g], o[x]);
            o[x] = Split::mfma(vh, pl[g], o[x]);
            o[x] = Split::mfma(vh, ph[g], o[x]);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          if constexpr (!careful) {  // a scale in which the sums of the finite ones stay finite
            float finite = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) finite = fmaxf(finite, fabsf(f[e]) < INFINITY ? fabsf(f[e]) : 0.f);
            v_top[x] = max(v_top[x], Split::exponent(wave_max_int(__float_as_int(finite))));
            if (v_exp[x] < v_top[x] - Split::kMost) scale_to(x, v_top[x] - Split::kMost);
          }
          const float by = Split::power(Split::kTop - v_exp[x]);
#pragma unroll
          for (int e = 0; e < 16; ++e)
            o[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(f[e] * by, s[0][e], o[x], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // step e takes keys 8 (e / 4) + 4 lh + e % 4: register e of s
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
          for (int x = 0; x < kO; ++x) {
            const float f = *reinterpret_cast<const float*>(
                all + (v_at ^ (x << 7) ^ ((e & 3) << 6) ^ (((e >> 2) & 1) << 5)) +
                (32 * u + 8 * (e >> 2) + (e & 3)) * kPitch);
            o[x] = __builtin_amdgcn_mfma_f32_32x32x2f32(f, s[u][e], o[x], 0, 0, 0);
          }
    }
  };

  // the tiles that some row of the workgroup may see
  int chunk = 0, tiles_seen = 0;
  unsigned long long todo = 0, any_word = 0, whole_word = 0, one_word = 0;
  auto sort_tiles = [&](const int4 k) __attribute__((always_inline)) {
    const int t = chunk * 64 + lane;
    const bool here = t >= lo && t < hi;
    const bool shared = prefixed && t < p_tiles;
    auto may_see = [&](const Range& r) { return here & (prefixed ? (shared & (r.dmax >= 0)) | (!shared & may_see_tile(k, r)) : may_see_tile(k, r)); };
    todo = __ballot(may_see(all_rows));
    if ((in_parts || kTeams > 1 || windowed) && parts > 1) {  // every parts-th of them
      const int number = tiles_seen + __popcll(todo & ((1ull << lane) - 1));
      tiles_seen += __popcll(todo);
      todo = __ballot(((todo >> lane) & 1) && number % parts == part);
    }
    any_word = __ballot(may_see(mine));
    const bool one = (k.x == k.y) & (mine.dmin == mine.dmax) & (k.x == mine.dmin);
    bool whole = one & ((t + 1 - p_tiles) * kTile <= k_len) & (k.w <= mine.omin);
    if (windowed) whole &= (k.z >= window_from(mine.omax)) | ((k.z >= 0) & (k.w < a.sinks));
    if (prefixed) whole = shared ? (t + 1) * kTile <= a.p.len : whole;
    whole_word = __ballot(here & whole);
    if (windowed || prefixed) one_word = __ballot(one | shared);
  };
  struct Next {
    int tile;
    bool any, whole, one;  // seen by some row of the wave; by all; by orders and the keys' end alone
  };
  auto next_tile = [&]() __attribute__((always_inline)) -> Next {
    while (todo == 0) {
      ++chunk;
      if (windowed)
        while (chunk * 64 < hi && !((chunks >> min(chunk, 63)) & 1)) ++chunk;
      if (chunk * 64 >= hi) return Next{-1, false, false, false};
      sort_tiles(summary_of(chunk * 64 + lane));
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    return Next{chunk * 64 + bit, (bool)((any_word >> bit) & 1), (bool)((whole_word >> bit) & 1), (bool)((one_word >> bit) & 1)};
  };

  auto walk = [&](auto careful_c) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[x][v] = 0.f;
    m_run = -INFINITY, l_run = 0.f, base = kShift, mixed_seen = false;
    if constexpr (kSplit) {
#pragma unroll
      for (int x = 0; x < kO; ++x) v_exp[x] = decltype(careful_c)::value ? Split::kTop : Split::kLeast, v_top[x] = Split::kLeast;
    }
    chunk = lo / 64, tiles_seen = 0;
    sort_tiles(decltype(careful_c)::value ? summary_of(lo / 64 * 64 + lane) : first_summary);
    Next now = next_tile();
    int buf = 2 * team;
    if (now.tile >= 0) load_tile(now.tile, buf);
    if constexpr (kWaves == 1 && kTeams == 1 && k16) {
      // A wave by itself keeps two tiles in flight: the one after the next is asked for as soon as this
      // one has been read, before its softmax.  At least 2 kLoads loads are younger than this
      // tile's.  16 tokens over 16384 keys, 32 heads on 8 of 128, bf16: 210 -> 200 us.  Not for teams
      // (12.9 -> 13.1 us; one CU's loads are what they wait for) nor fp32 (the same).
      Next then = now.tile >= 0 ? next_tile() : now;
      if (then.tile >= 0) load_tile(then.tile, buf ^ 1);
      while (now.tile >= 0) {
        const Next after = then.tile >= 0 ? next_tile() : then;
        if (then.tile >= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const auto read = [&]() __attribute__((always_inline)) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (after.tile >= 0) load_tile(after.tile, buf);
        };
        if (now.any) attend(buf, now.tile, now.whole, now.one, careful_c, read);
        if (decltype(careful_c)::value || !now.any) read();
        buf ^= 1;
        now = then, then = after;
      }
      return;
    }
    while (now.tile >= 0) {
      const Next then = next_tile();
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of tile `now` is in LDS
      if constexpr (kTeams > 1) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      else __syncthreads();  // everyone's is, and everyone is done with the other buffer
      if (then.tile >= 0) load_tile(then.tile, buf ^ 1);
      if (now.any) attend(buf, now.tile, now.whole, now.one, careful_c, [] {});
      buf ^= 1;
      now = then;
    }
  };
  walk(std::integral_constant<bool, false>{});
  // 0 * V of an unseen key is NaN where V is not finite: then all over again, with care
  bool bad = false;
  if (mixed_seen && live) {
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) bad |= !(fabsf(o[x][v]) < INFINITY);
  }
  // also the barrier before the buffers are filled again
  if (kTeams > 1 ? __any(bad) : __syncthreads_or(bad)) walk(std::integral_constant<bool, true>{});

  l_run = halves_sum(l_run);
  if constexpr (kSplit) {  // without the probabilities' factor: V up to the type's end, as the other fp32 kernels bear
    l_run = __builtin_ldexpf(l_run, -(int)kShift);
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[x][v] = __builtin_ldexpf(o[x][v], v_exp[x] - Split::kTop - (int)kShift);
  }
  if constexpr (kTeams > 1) {
    // each team's (maximum, sum) and output in its own place, then all of them in order
    constexpr int kPlace = kPart;  // floats of a team's place: four tiles' bytes
    static_assert(32 * kD + 64 <= kPlace, "a team's output fits its place");
    float* places = reinterpret_cast<float*>(&staged[0][0]);
    float* mine_at = places + team * kPlace;
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(mine_at + lq * kD + 32 * x + 8 * g + 4 * lh) =
            make_float4(o[x][4 * g], o[x][4 * g + 1], o[x][4 * g + 2], o[x][4 * g + 3]);
    if (lh == 0) {
      mine_at[32 * kD + 2 * lq] = live ? m_run * to_log2 : -INFINITY;
      mine_at[32 * kD + 2 * lq + 1] = live ? l_run : 0.f;
    }
    __syncthreads();
    for (int e = tid; e < a.rows * (d / 4); e += kTeams * kWave) {
      const int r = e / (d / 4), at = e % (d / 4) * 4;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < kTeams; ++i) top = fmaxf(top, places[i * kPlace + 32 * kD + 2 * r]);
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kTeams; ++i) {
        const float* from = places + i * kPlace;
        const float l = from[32 * kD + 2 * r + 1];
        if (l == 0.f) continue;  // nothing seen (a part whose scores are NaN has its sum NaN)
        const float w = __builtin_amdgcn_exp2f(from[32 * kD + 2 * r] - top);
        const float4 p = *reinterpret_cast<const float4*>(from + r * kD + at);
        sum = fmaf(w, l, sum);
        y.x = fmaf(w, p.x, y.x), y.y = fmaf(w, p.y, y.y), y.z = fmaf(w, p.z, y.z), y.w = fmaf(w, p.w, y.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int t = (int)((uint32_t)r / (uint32_t)a.group), h = kvh * a.group + (r - t * a.group);
      typedef T Four __attribute__((ext_vector_type(4)));
      *reinterpret_cast<Four*>(static_cast<T*>(c.out) + b * c.o_sb + (long long)t * c.o_st + h * c.o_sh + at) =
          Four{(T)(y.x * inv), (T)(y.y * inv), (T)(y.z * inv), (T)(y.w * inv)};
    }
    return;
  }
  if (!inside) return;
  // register v of block x holds channel 32 x + 8 (v / 4) + 4 lh + v % 4
  if (in_parts ? parts == 1 : a.splits == 1 && !(prefixed && a.partial)) {
    const bool empty = !live || l_run == 0.f;
    const float inv = 1.f / l_run;
    T* orow = static_cast<T*>(c.out) + b * c.o_sb + (long long)token * c.o_st + head * c.o_sh;
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * x + 8 * g + 4 * lh;
        typedef T Four __attribute__((ext_vector_type(4)));
        Four y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = empty ? (T)0.f : (T)(o[x][4 * g + i] * inv);
        if (at < d) *reinterpret_cast<Four*>(orow + at) = y;
      }
  } else {
    const long long at_row = !in_parts ? ((long long)bh * a.rows + row) * a.splits + split
                                       : ((long long)bh * a.jobs + job) * kRowTile + row % kRowTile;
    if (lh == 0) {
      a.part_ml[2 * at_row] = live ? m_run * to_log2 : -INFINITY;
      a.part_ml[2 * at_row + 1] = live ? l_run : 0.f;
    }
    float* prow = a.part_o + at_row * d;
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = 32 * x + 8 * g + 4 * lh;
        const float4 y = make_float4(o[x][4 * g], o[x][4 * g + 1], o[x][4 * g + 2], o[x][4 * g + 3]);
        if (at < d) *reinterpret_cast<float4*>(prow + at) = live ? y : make_float4(0.f, 0.f, 0.f, 0.f);
      }
  }
}

#define MUSC_MASKED_ATTENTION_BOUNDS \
  __launch_bounds__(kWaves * kTeams * kWave, kWaves == 1 ? 1 : kD == 64 && kDtype != MUSC_DTYPE_F32 ? 3 : 2)
template <int kDtype, int kD, int kWaves, int kTeams, int kMode>
__global__ MUSC_MASKED_ATTENTION_BOUNDS void masked_attention_kernel(const Args a) {
  attention_of_block<kDtype, kD, kWaves, kTeams, kMode>(a, blockIdx.x, gridDim.x);
}
// The same with the work of two calls side by side, the second's workgroups after the first's (whose number
// is a multiple of the XCDs).
template <int kDtype, int kD, int kWaves, int kTeams, int kMode>
__global__ MUSC_MASKED_ATTENTION_BOUNDS void prefixed_attention_kernel(const TwoArgs two) {
  const bool second = blockIdx.x >= two.first_blocks;
  const uint32_t before = second ? two.first_blocks : 0, blocks = second ? gridDim.x - before : two.first_blocks;
  attention_of_block<kDtype, kD, kWaves, kTeams, kMode>(second ? two.second : two.first, blockIdx.x - before, blocks);
}

// Joins the splits of a row, in their order: four waves per row, each every fourth split with two
// channels per lane, then the four in order.
template <int kDtype>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  typedef typename Type<kDtype>::T T;
  __shared__ float weight[kMaxSplits], tops[4], sums[4];
  __shared__ float2 parts[4][kWave];
  const musc_masked_attention& c = a.c;
  const long long r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int splits = a.splits;
  // the largest of the maxima, each split's factor and the sum; a part without keys has sum 0
  // (one whose scores are NaN has its sum NaN)
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + r * splits;
  const float2 mine = tid < splits ? ml[tid] : make_float2(-INFINITY, 0.f);
  const float top_here = wave_max(mine.x);
  if (lane == 0) tops[wave] = top_here;
  __syncthreads();
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float w = mine.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(mine.x - top);
  if (tid < splits) weight[tid] = w;
  const float sum_here = wave_sum(mine.y == 0.f ? 0.f : w * mine.y);
  if (lane == 0) sums[wave] = sum_here;
  __syncthreads();
  const float sum = sums[0] + sums[1] + sums[2] + sums[3];
  const bool ok = 2 * lane < c.d;
  const float* at = a.part_o + r * splits * c.d + (ok ? 2 * lane : 0);
  float2 y = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int s = wave; s < splits; s += 4) {
    const float2 p = *reinterpret_cast<const float2*>(at + (long long)s * c.d);
    const float f = weight[s];
    if (f != 0.f) y.x = fmaf(f, p.x, y.x), y.y = fmaf(f, p.y, y.y);
  }
  parts[wave][lane] = y;
  __syncthreads();
  if (wave != 0 || !ok) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) y.x += parts[i][lane].x, y.y += parts[i][lane].y;
  const float inv = 1.f / sum;
  const long long bh = r / a.rows;
  const int row = (int)(r % a.rows), token = row / a.group;
  const int head = (int)(bh % c.kv_heads) * a.group + row % a.group;
  typedef T Two __attribute__((ext_vector_type(2)));
  Two out;
  out[0] = sum == 0.f ? (T)0.f : (T)(y.x * inv);
  out[1] = sum == 0.f ? (T)0.f : (T)(y.y * inv);
  T* orow = static_cast<T*>(c.out) + (bh / c.kv_heads) * c.o_sb + (long long)token * c.o_st + head * c.o_sh;
  *reinterpret_cast<Two*>(orow + 2 * lane) = out;
}

// Joins the parts of windowed and prefixed attention's rows, a.splits and then a.more_splits of them, in
// their order: kShare waves a row, each every kShare-th part with two channels per lane, then those in
// order.  The first eight parts of a wave are asked for before their factors are formed.  Four waves for
// few rows, else one (4160 rows of 18 parts, fp32: 9 us with four, 6 with one).
template <int kDtype, bool kByKeyHead, int kShare>
__global__ __launch_bounds__(256) void join_rows_kernel(const Args a, const long long all_rows) {
  typedef typename Type<kDtype>::T T;
  __shared__ float2 shared[kShare > 1 ? 4 : 1][kWave];
  const musc_masked_attention& c = a.c;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), part = wave % kShare;
  const long long r = (long long)blockIdx.x * (4 / kShare) + wave / kShare;
  if (r >= all_rows) return;  // whole workgroups with kShare > 1
  const int splits = a.splits, all = splits + a.more_splits;
  const bool ok = 2 * lane < c.d;
  const int at = ok ? 2 * lane : 0;
  const float *first_o = a.part_o + r * splits * c.d + at, *more_o = a.more_o + (r * a.more_splits - splits) * c.d + at;
  auto load = [&](int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const float2*>((s < splits ? first_o : more_o) + (long long)s * c.d);
  };
  constexpr int kBatch = 8;
  float2 p[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) p[i] = load(min(part + i * kShare, all - 1));
  // the largest of the maxima, each part's factor and the sum; a part without keys has sum 0 (one whose
  // scores are NaN has its sum NaN)
  constexpr int kPer = kMaxSplits / kWave;
  float w[kPer], l[kPer], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = i * kWave + lane;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (s < splits) ml = reinterpret_cast<const float2*>(a.part_ml)[r * splits + s];
    else if (s < all) ml = reinterpret_cast<const float2*>(a.more_ml)[r * a.more_splits + s - splits];
    w[i] = ml.x, l[i] = ml.y;
    top = fmaxf(top, ml.x);
  }
  top = wave_max(top);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    w[i] = l[i] == 0.f ? 0.f : __builtin_amdgcn_exp2f(w[i] - top);
    sum += l[i] == 0.f ? 0.f : w[i] * l[i];
  }
  sum = wave_sum(sum);
  float2 y = make_float2(0.f, 0.f);
  for (int from = part; from < all; from += kBatch * kShare) {
    if (from != part) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) p[i] = load(min(from + i * kShare, all - 1));
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int s = from + i * kShare;
      const float of = s < kWave ? w[0] : s < 2 * kWave ? w[1] : s < 3 * kWave ? w[2] : w[3];
      const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(of), s % kWave));
      if (s < all && f != 0.f) y.x = fmaf(f, p[i].x, y.x), y.y = fmaf(f, p[i].y, y.y);
    }
  }
  if constexpr (kShare > 1) {
    shared[wave][lane] = y;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 1; i < kShare; ++i) y.x += shared[i][lane].x, y.y += shared[i][lane].y;
  }
  if (!ok) return;
  const float inv = 1.f / sum;
  const int rows = c.q_len * a.group;  // of a batch entry and key head
  const long long bh = r / rows;
  const int row = (int)(r % rows), token = row / a.group;
  const int b = (int)(kByKeyHead ? bh % c.batch : bh / c.kv_heads);
  const int head = (int)(kByKeyHead ? bh / c.batch : bh % c.kv_heads) * a.group + row % a.group;
  typedef T Two __attribute__((ext_vector_type(2)));
  Two out;
  out[0] = sum == 0.f ? (T)0.f : (T)(y.x * inv);
  out[1] = sum == 0.f ? (T)0.f : (T)(y.y * inv);
  *reinterpret_cast<Two*>(static_cast<T*>(c.out) + b * c.o_sb + (long long)token * c.o_st + head * c.o_sh + 2 * lane) = out;
}
template <int kDtype, bool kByKeyHead>
void launch_join(const Args& a, hipStream_t stream) {
  const long long rows = (long long)a.c.batch * a.c.kv_heads * a.c.q_len * a.group;
  if (rows <= 1024)
    hipLaunchKernelGGL((join_rows_kernel<kDtype, kByKeyHead, 4>), dim3((unsigned)rows), dim3(256), 0, stream, a, rows);
  else
    hipLaunchKernelGGL((join_rows_kernel<kDtype, kByKeyHead, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a, rows);
}

// Joins the parts of the row tiles that were done in parts, in their order: a workgroup per row
// tile, four channels of a row per thread.
template <int kDtype>
__global__ __launch_bounds__(256) void join_parts_kernel(const Args a) {
  typedef typename Type<kDtype>::T T;
  const musc_masked_attention& c = a.c;
  const int tile = blockIdx.x % a.row_tiles, bh = blockIdx.x / a.row_tiles, b = bh / c.kv_heads;
  const int entry = c.schedule[b * c.schedule_sb + kScheduleHead + 2 * a.row_tiles + tile];
  const int job = entry & 0xffffff, parts = min((entry >> 24) & 15, kMaxParts);
  if (parts <= 1 || job + parts > a.jobs) return;
  const int first_row = tile * kRowTile, rows = min(kRowTile, a.rows - first_row);
  const int of_row = c.d / 4;
  const long long first = ((long long)bh * a.jobs + job) * kRowTile;
  for (int e = threadIdx.x; e < rows * of_row; e += 256) {
    const int r = e / of_row, at = e % of_row * 4;
    float m[kMaxParts], l[kMaxParts], top = -INFINITY;
    float4 p[kMaxParts];
#pragma unroll
    for (int i = 0; i < kMaxParts; ++i) {
      m[i] = -INFINITY, l[i] = 0.f, p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < parts) {
        const long long from = first + i * kRowTile + r;
        const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[from];
        m[i] = ml.x, l[i] = ml.y;
        p[i] = *reinterpret_cast<const float4*>(a.part_o + from * c.d + at);
      }
      top = fmaxf(top, m[i]);
    }
    float sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kMaxParts; ++i) {
      if (l[i] == 0.f) continue;  // nothing seen (a part whose scores are NaN has its sum NaN)
      const float w = __builtin_amdgcn_exp2f(m[i] - top);
      sum = fmaf(w, l[i], sum);
      y.x = fmaf(w, p[i].x, y.x), y.y = fmaf(w, p[i].y, y.y), y.z = fmaf(w, p[i].z, y.z), y.w = fmaf(w, p[i].w, y.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int row = first_row + r, token = row / a.group;
    const int head = bh % c.kv_heads * a.group + row % a.group;
    typedef T Four __attribute__((ext_vector_type(4)));
    const Four out = {(T)(y.x * inv), (T)(y.y * inv), (T)(y.z * inv), (T)(y.w * inv)};
    *reinterpret_cast<Four*>(static_cast<T*>(c.out) + b * c.o_sb + (long long)token * c.o_st + head * c.o_sh + at) = out;
  }
}

// Few rows, rows in parts, or a large cap.
template <int kDtype, int kD, int kMode>
void launch_special(const Args& a, int waves, const dim3& grid, hipStream_t stream) {
  constexpr int kTeams = teams_of((kD <= 64 ? 64 : 128) * (kDtype == MUSC_DTYPE_F32 ? 4 : 2));
  if (a.teams > 1)
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 1, kTeams, kMode>), grid, dim3(kTeams * kWave), 0, stream, a);
  else if (waves == 1)
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 1, 1, kMode>), grid, dim3(kWave), 0, stream, a);
  else if (a.in_parts)
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, kMode | kInParts>), grid, dim3(4 * kWave), 0, stream, a);
  else if constexpr ((kMode & kLargeCap) != 0)
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, kMode>), grid, dim3(4 * kWave), 0, stream, a);
}

template <int kDtype, int kD>
void launch(const Args& a, int waves, hipStream_t stream) {
  const dim3 grid((unsigned)align_up((size_t)a.units, kXcds));
  const int mode = (a.c.cap > 0.f ? kCapped : 0) | (a.c.axes ? kBiased : 0);
  constexpr int kWide = kD <= 64 ? 64 : 128;
  if constexpr (kDtype != MUSC_DTYPE_F32) {
    if (a.c.cap > kSmallCap) return launch_special<kDtype, kWide, kEither | kLargeCap>(a, waves, grid, stream);
  }
  if (waves == 1 || a.in_parts) {
    if (mode == 0) launch_special<kDtype, kWide, 0>(a, waves, grid, stream);
    else launch_special<kDtype, kWide, kEither>(a, waves, grid, stream);
  } else if (mode == 0) {
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, 0>), grid, dim3(4 * kWave), 0, stream, a);
  } else if (mode == kCapped) {
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, kCapped>), grid, dim3(4 * kWave), 0, stream, a);
  } else if (mode == kBiased) {
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, kBiased>), grid, dim3(4 * kWave), 0, stream, a);
  } else {
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, 4, 1, kCapped | kBiased>), grid, dim3(4 * kWave), 0, stream, a);
  }
}

// Windows and shared prefixes (kExtra): the same kernels with that mode, no parts of row tiles, and one
// kernel for caps and biases (2 % over one for each: 24 frames of 256 tokens with a bias 91 us and 89).
template <int kDtype, int kD, int kWaves, int kTeams, int kMode>
void launch_one(const Args& a, const Args* more, hipStream_t stream) {
  const size_t blocks = align_up((size_t)a.units, kXcds), all = blocks + (more ? align_up((size_t)more->units, kXcds) : 0);
  if constexpr ((kMode & kPrefixed) != 0) {
    const TwoArgs two{a, more ? *more : a, (uint32_t)blocks};
    hipLaunchKernelGGL((prefixed_attention_kernel<kDtype, kD, kWaves, kTeams, kMode>), dim3((unsigned)all),
                       dim3(kWaves * kTeams * kWave), 0, stream, two);
  } else {
    hipLaunchKernelGGL((masked_attention_kernel<kDtype, kD, kWaves, kTeams, kMode>), dim3((unsigned)all),
                       dim3(kWaves * kTeams * kWave), 0, stream, a);
  }
}
template <int kDtype, int kD, int kMode>
void launch_few(const Args& a, const Args* more, hipStream_t stream) {
  constexpr int kTeams = teams_of((kD <= 64 ? 64 : 128) * (kDtype == MUSC_DTYPE_F32 ? 4 : 2));
  if (a.teams > 1) launch_one<kDtype, kD, 1, kTeams, kMode>(a, more, stream);
  else launch_one<kDtype, kD, 1, 1, kMode>(a, more, stream);
}
// Four waves.
template <int kDtype, int kD, int kMode>
void launch_many(const Args& a, const Args* more, hipStream_t stream) {
  if constexpr (kDtype != MUSC_DTYPE_F32 && (kMode & kPrefixed) != 0) {
    if (a.two_numbers) return launch_one<kDtype, kD, 4, 1, kMode | kTwoNumbers>(a, more, stream);
  }
  launch_one<kDtype, kD, 4, 1, kMode>(a, more, stream);
}
template <int kDtype, int kD, int kExtra>
void launch_extra(const Args& a, const Args* more, int waves, hipStream_t stream) {
  const bool plain = !(a.c.cap > 0.f) && !a.c.axes;
  constexpr int kWide = kD <= 64 ? 64 : 128;
  if constexpr (kDtype != MUSC_DTYPE_F32) {
    if (a.c.cap > kSmallCap) {
      if (waves == 1) launch_few<kDtype, kWide, kEither | kLargeCap | kExtra>(a, more, stream);
      else launch_many<kDtype, kWide, kEither | kLargeCap | kExtra>(a, more, stream);
      return;
    }
  }
  if (waves == 1) {
    if (plain) launch_few<kDtype, kWide, kExtra>(a, more, stream);
    else launch_few<kDtype, kWide, kEither | kExtra>(a, more, stream);
  } else if (plain) {
    launch_many<kDtype, kD, kExtra>(a, more, stream);
  } else {
    launch_many<kDtype, kD, kEither | kExtra>(a, more, stream);
  }
}
template <int kDtype, int kExtra>
void launch_extra(const Args& a, const Args* more, int waves, hipStream_t stream) {
  if (a.c.d <= 64) launch_extra<kDtype, 64, kExtra>(a, more, waves, stream);
  else if (a.c.d <= 96) launch_extra<kDtype, 96, kExtra>(a, more, waves, stream);
  else launch_extra<kDtype, 128, kExtra>(a, more, waves, stream);
}
template <int kDtype>
void launch_windowed(const Args& a, int waves, hipStream_t stream) {
  launch_extra<kDtype, kWindowed>(a, nullptr, waves, stream);
  if (a.splits > 1) launch_join<kDtype, false>(a, stream);
}
// more: the entries' own keys, beside all rows over the prefix.
template <int kDtype>
void launch_prefixed(const Args& a, const Args* more, int waves, hipStream_t stream) {
  launch_extra<kDtype, kPrefixed>(a, more, waves, stream);
  if (a.splits > 1 || a.stacked) {
    Args both = a;
    if (more) both.more_splits = more->splits, both.more_ml = more->part_ml, both.more_o = more->part_o;
    launch_join<kDtype, true>(both, stream);
  }
}

template <int kDtype>
void launch_all(const Args& a, int waves, hipStream_t stream) {
  if (a.c.d <= 64) launch<kDtype, 64>(a, waves, stream);
  else if (a.c.d <= 96) launch<kDtype, 96>(a, waves, stream);
  else launch<kDtype, 128>(a, waves, stream);
  if (a.in_parts)
    hipLaunchKernelGGL((join_parts_kernel<kDtype>), dim3((unsigned)(a.units / a.jobs * a.row_tiles)), dim3(256), 0, stream, a);
  if (a.splits > 1) {
    const long long rows = (long long)a.c.batch * a.c.kv_heads * a.rows;
    hipLaunchKernelGGL((join_kernel<kDtype>), dim3((unsigned)rows), dim3(256), 0, stream, a);
  }
}

}  // namespace mattn
}  // namespace musc
