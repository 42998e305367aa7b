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
constexpr int kCapped = 1, kBiased = 2, kInParts = 4, kEither = 8, kLargeCap = 16;
template <int kDtype, int kD, int kWaves, int kTeams, int kMode>
__global__ __launch_bounds__(kWaves * kTeams * kWave, kWaves == 1 ? 1 : kD == 64 && kDtype != MUSC_DTYPE_F32 ? 3 : 2) void masked_attention_kernel(
    const Args a) {
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
  __shared__ __attribute__((aligned(1024))) char staged[2 * kTeams][2 * kPart];
  __shared__ __attribute__((aligned(16))) int docs_s[2 * kTeams][64], ords_s[2 * kTeams][64];
  __shared__ float pos_s[2 * kTeams][64 * kMaxAxes];
  __shared__ Range ranges[kWaves];

  const musc_masked_attention& c = a.c;
  // uniform numbers in scalar registers (the divisions leave them in vector ones)
  const auto uniform = [](long long x) { return __builtin_amdgcn_readfirstlane((int)x); };
  uint32_t split, job, bh;
  if (a.heads_at_once) {
    // one XCD works on heads_at_once heads together, row tile by row tile (the longest first)
    const uint32_t per_xcd = (uint32_t)(c.batch * c.kv_heads) / kXcds, local = blockIdx.x / kXcds;
    const uint32_t of_group = (uint32_t)(a.heads_at_once * a.jobs * a.splits);
    const uint32_t group = uniform(local / of_group), in_group = local - group * of_group;
    const uint32_t first = group * a.heads_at_once, at_once = min((uint32_t)a.heads_at_once, per_xcd - first);
    const uint32_t rest = uniform(in_group / a.splits);
    split = in_group - rest * a.splits;
    job = uniform(rest / at_once);
    bh = blockIdx.x % kXcds * per_xcd + first + (rest - job * at_once);
  } else {
    const uint32_t unit = (blockIdx.x % kXcds) * (gridDim.x / kXcds) + blockIdx.x / kXcds;
    if (unit >= (uint32_t)a.units) return;
    const uint32_t rest = uniform(unit / a.splits);
    split = unit - rest * a.splits;
    bh = uniform(rest / a.jobs);
    job = rest - bh * a.jobs;
  }
  const int b = uniform(bh / c.kv_heads), kvh = bh - b * c.kv_heads;
  const int tid = threadIdx.x, lane = tid % kWave;
  const int team = kTeams > 1 ? __builtin_amdgcn_readfirstlane(tid / kWave) : 0;
  const int wave = kTeams > 1 ? 0 : __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lq = lane & 31, lh = lane >> 5;

  // tiles of this split, 64 sorted at a time by the keys' summary; the first 64 are asked for now
  const int lo = uniform((long long)a.key_tiles * split / a.splits);
  const int hi = uniform((long long)a.key_tiles * (split + 1) / a.splits);
  const int4* summary = c.k_summary ? reinterpret_cast<const int4*>(c.k_summary) + b * c.k_summary_sb : nullptr;
  auto summary_of = [&](int t) __attribute__((always_inline)) {
    int4 k = make_int4(0, 0, 0, 0);
    if (summary && t >= lo && t < hi) {
      k = summary[(long long)t * kSub];
      if (kSub > 1 && t * kSub + 1 < a.summaries) {
        const int4 n = summary[(long long)t * kSub + 1];
        k = make_int4(min(k.x, n.x), max(k.y, n.y), min(k.z, n.z), max(k.w, n.w));
      }
    }
    return k;
  };
  const int4 first_summary = summary_of(lo / 64 * 64 + lane);

  // the row tile, or the part of its keys, that the schedule names; without one later rows first:
  // with an order of tokens they see more keys, and the longest work should not start last
  constexpr bool in_parts = (kMode & kInParts) != 0;
  int tile_of_rows = a.row_tiles - 1 - (int)job, part = team, parts = kTeams;
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
  const int token = inside ? (int)((uint32_t)row / (uint32_t)a.group) : 0;
  const int head = kvh * a.group + (inside ? row - token * a.group : 0);
  const int d = c.d, k_len = c.k_len, axes = kMode & (kBiased | kEither) ? c.axes : 0;

  // this row's document and order (rows outside the tensor read token 0's), its Q and positions,
  // all asked for before any is used
  int qdoc = 0, qord = 0;
  if (c.q_documents) qdoc = c.q_documents[b * c.q_tokens_sb + token];
  if (c.q_order) qord = c.q_order[b * c.q_tokens_sb + token];
  const T* qrow = static_cast<const T*>(c.q) + b * c.q_sb + (long long)token * c.q_st + head * c.q_sh;
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
      qpos[x] = c.q_positions[b * c.q_positions_sb + (long long)token * axes + x];
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
  const uint32_t k_row = (uint32_t)(c.k_st * (long long)sizeof(T)), v_row = (uint32_t)(c.v_st * (long long)sizeof(T));
  const uint32_t staged_at = (uint32_t)(size_t)(lds_void*)&staged[0][0] + wave * 1024;
  constexpr int kRows = 64 / kPlaces;  // rows of a load
  const int row_bytes = d * (int)sizeof(T);
  auto load_tile = [&](int tile, int buf) __attribute__((always_inline)) {
    const int first = tile * kTile, rem = min(k_len - first, kTile), mine = wave * kRows;
    const uint32_t to = __builtin_amdgcn_readfirstlane(staged_at + buf * 2 * kPart);
    const char* kt = kbase + (unsigned long long)(uint32_t)(first + mine) * k_row;
    const char* vt = vbase + (unsigned long long)(uint32_t)(first + mine) * v_row;
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
      if (c.k_documents)
        load_to_lds_4(&docs_s[buf][0], lane * 4,
                      resource(c.k_documents + b * c.k_tokens_sb + first, rem * 4));
      if (c.k_order)
        load_to_lds_4(&ords_s[buf][0], lane * 4,
                      resource(c.k_order + b * c.k_tokens_sb + first, rem * 4));
      if (axes) {
        const int4v rp = resource(c.k_positions + b * c.k_positions_sb + (long long)first * axes, rem * axes * 4);
#pragma unroll
        for (int x = 0; x < kMaxAxes; ++x)
          if (x < axes) load_to_lds_4(&pos_s[buf][64 * x], (64 * x + lane) * 4, rp);
      }
    }
  };

  floatx16 o[kO];
  float m_run, l_run;  // running maximum (raw) and sum of this half's keys
  float base;          // exponent of a score: raw * to_log2 + base
  bool mixed_seen;

  // one staged tile; whole: every row sees every key.  careful: in a mixed tile, products
  // of keys that a row does not see are left out one by one (their V may be infinite or NaN)
  auto attend = [&](int buf, int tile, bool whole, auto careful_c, auto read) __attribute__((always_inline)) {
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
          s[u][v] = by_exponential ? __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(x)) : tanhf(x);
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
      const int rem = k_len - tile * kTile;
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
      base = Ty::kShift - (m_run == -INFINITY ? 0.f : m_run * to_log2);
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[u][v] = __builtin_amdgcn_exp2f(fmaf(s[u][v], to_log2, base));
    TVec p[2 * kSub];
    if constexpr (k16) {
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
            if (u == u0 && v == v0) pr = (float)(T)s[u][v];
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
        for (int x = 0; x < kO; ++x)
          o[x] = Ty::mfma(__builtin_bit_cast(TVec, careful ? read_v(mm, x) : vf[careful ? 0 : mm][careful ? 0 : x]), p[mm], o[x]);
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
  unsigned long long todo = 0, any_word = 0, whole_word = 0;
  auto sort_tiles = [&](const int4 k) __attribute__((always_inline)) {
    const int t = chunk * 64 + lane;
    const bool here = t >= lo && t < hi;
    auto may_see = [&](const Range& r) {
      return here && k.y >= 0 && k.x <= r.dmax && k.y >= r.dmin && k.z <= r.omax;
    };
    todo = __ballot(may_see(all_rows));
    if ((in_parts || kTeams > 1) && parts > 1) {  // every parts-th of them
      const int number = tiles_seen + __popcll(todo & ((1ull << lane) - 1));
      tiles_seen += __popcll(todo);
      todo = __ballot(((todo >> lane) & 1) && number % parts == part);
    }
    any_word = __ballot(may_see(mine));
    whole_word = __ballot(here && k.x == k.y && mine.dmin == mine.dmax && k.x == mine.dmin && k.w <= mine.omin &&
                          (t + 1) * kTile <= k_len);
  };
  struct Next {
    int tile;
    bool any, whole;
  };
  auto next_tile = [&]() __attribute__((always_inline)) -> Next {
    while (todo == 0) {
      ++chunk;
      if (chunk * 64 >= hi) return Next{-1, false, false};
      sort_tiles(summary_of(chunk * 64 + lane));
    }
    const int bit = __builtin_ctzll(todo);
    todo &= todo - 1;
    return Next{chunk * 64 + bit, (bool)((any_word >> bit) & 1), (bool)((whole_word >> bit) & 1)};
  };

  auto walk = [&](auto careful_c) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < kO; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[x][v] = 0.f;
    m_run = -INFINITY, l_run = 0.f, base = Ty::kShift, mixed_seen = false;
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
        if (now.any) attend(buf, now.tile, now.whole, careful_c, read);
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
      if (now.any) attend(buf, now.tile, now.whole, careful_c, [] {});
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
  if (in_parts ? parts == 1 : a.splits == 1) {
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
