// Masked attention's C entry points: the keys' summary, the order of self-attention's row
// tiles, and the launch of masked_attention_kernel.hpp's kernels.
#include "masked_attention.hpp"

namespace musc {
namespace mattn {

// Per 32 keys: smallest and largest document (negative ones count as -1), smallest and largest
// order of the keys that have a document.  One wave handles two groups of 32.
__global__ __launch_bounds__(256) void token_summary_kernel(const int* __restrict__ documents,
                                                            const int* __restrict__ order, int batch, int t,
                                                            int groups, int4* __restrict__ summary) {
  const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) / kSummaryKeys;
  if (g >= (long long)batch * groups) return;  // whole halves of a wave; the shuffles stay inside them
  const int b = (int)(g / groups), first = (int)(g % groups) * kSummaryKeys;
  const int key = first + threadIdx.x % kSummaryKeys;
  int doc = -1, ord = 0;
  if (key < t) {
    doc = max(documents[(long long)b * t + key], -1);
    if (order) ord = order[(long long)b * t + key];
  }
  int4 s = make_int4(doc, doc, doc < 0 ? 0x7fffffff : ord, doc < 0 ? (int)0x80000000 : ord);
#pragma unroll
  for (int off = kSummaryKeys / 2; off >= 1; off >>= 1) {
    s.x = min(s.x, __shfl_xor(s.x, off, kSummaryKeys));
    s.y = max(s.y, __shfl_xor(s.y, off, kSummaryKeys));
    s.z = min(s.z, __shfl_xor(s.z, off, kSummaryKeys));
    s.w = max(s.w, __shfl_xor(s.w, off, kSummaryKeys));
  }
  if (threadIdx.x % kSummaryKeys == 0) summary[g] = s;
}

// Schedules of self-attention for 1, 2, 4 and 8 query heads per key head, one after the other,
// a block (see schedule_block) per batch entry.
struct Schedule {
  int batch, t, groups;
  int tiles[4];        // row tiles
  long long first[5];  // (batch entry, row tile) pairs before this number of heads
  long long at[4];     // first int of its blocks
  __device__ __forceinline__ int which(long long i) const { return (i >= first[1]) + (i >= first[2]) + (i >= first[3]); }
};

// Work of each row tile: the groups of 32 keys that its rows may see; and the document's start or end
// within it whose two sides have the least work each, if that is at most 3/4.  One wave per tile.
__global__ __launch_bounds__(kWave) void row_work_kernel(const int* __restrict__ documents, const int* __restrict__ order,
                                                         const int4* __restrict__ summary, const Schedule s,
                                                         int* __restrict__ out) {
  const int w = s.which(blockIdx.x), lane = threadIdx.x;
  const int i = (int)(blockIdx.x - s.first[w]), b = i / s.tiles[w], tile = i % s.tiles[w];
  const int first = tile * (kRowTile >> w), last = min(first + (kRowTile >> w), s.t) - 1;
  int* block = out + s.at[w] + b * schedule_block(s.tiles[w]);
  const int* docs = documents + (long long)b * s.t;
  const int4* keys = summary + (long long)b * s.groups;
  // groups that some token of from .. to - 1 may see
  auto work = [&](int from, int to) {
    Range r = {0x7fffffff, -1, 0x7fffffff, (int)0x80000000};
    for (int k = from + lane; k < to; k += kWave) {
      const int doc = docs[k], ord = order ? order[(long long)b * s.t + k] : 0;
      if (doc < 0) continue;
      r = Range{min(r.dmin, doc), max(r.dmax, doc), min(r.omin, ord), max(r.omax, ord)};
    }
    r = Range{wave_min_int(r.dmin), wave_max_int(r.dmax), wave_min_int(r.omin), wave_max_int(r.omax)};
    int count = 0;
    for (int g = lane; g < s.groups; g += kWave) {
      const int4 k = keys[g];
      count += k.y >= 0 && k.x <= r.dmax && k.y >= r.dmin && k.z <= r.omax;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) count += __shfl_xor(count, off, kWave);
    return count;
  };
  const int count = work(first, last + 1);
  // the end of the first document and the start of the last one: where a cut may halve the work
  int ends = last + 1, starts = first;
  for (int k = first + lane; k <= last; k += kWave) {
    if (docs[k] != docs[first]) ends = min(ends, k);
    if (docs[k] != docs[last]) starts = max(starts, k + 1);
  }
  ends = wave_min_int(ends), starts = wave_max_int(starts);
  int cut = 0, least = count * 3 / 4;
  if (ends <= last)
    for (int i = 0; i < (ends == starts ? 1 : 2); ++i) {
      const int at = i == 0 ? ends : starts, before = work(first, at), from = work(at, last + 1);
      if (max(before, from) > least) continue;
      least = max(before, from);
      cut = (at - first) << w | before << 7 | from << 17;
    }
  if (lane == 0) block[kScheduleHead + 3 * s.tiles[w] + schedule_jobs(s.tiles[w]) + tile] = cut;
  if (lane == 0) block[kScheduleHead + tile] = count;
}

// The row tiles by their work, most first (later ones first where it is the same): whole, and as
// jobs, where a tile of more than 5/4 of the mean work is listed in up to 8 parts, by the work of a
// part.  At most 9/5 n jobs.  And in pieces: the tiles of the most work, above the mean and n / 4 of them
// at most, cut where row_work_kernel found it worth while.
// Every row tile finds its places by looking at all of them in LDS: 1024 tiles, 1024 threads.  A
// schedule is shared by `slices` workgroups, which all form the same numbers and write their own tiles'.
constexpr int kMostTiles = MUSC_SCHEDULE_MAX_TOKENS * 8 / kRowTile;
__global__ __launch_bounds__(1024) void row_order_kernel(const Schedule s, int slices, int* __restrict__ out) {
  static_assert(kMostTiles <= 1024, "one row tile per thread");
  // Per tile, keys that are larger for what comes first: work << 10 | tile (whole), then (work of a part
  // << 10 | tile) << 3 | parts - 1, then the whole key's form for the tile's pieces (-1: not cut).
  __shared__ int4 keys[kMostTiles];
  __shared__ long long sums[16];
  __shared__ int counts[16], cuts_here[16];
  const int slice = blockIdx.x % slices, w = blockIdx.x / slices % 4, b = blockIdx.x / slices / 4;
  const int n = s.tiles[w], j = threadIdx.x, lane = j % kWave, wave = j / kWave;
  int* block = out + s.at[w] + b * schedule_block(n);
  const int x = j < n ? block[kScheduleHead + j] : 0;
  const double total = wave_sum((double)x);  // whole numbers below 2^53
  if (lane == 0) sums[wave] = (long long)total;
  __syncthreads();
  long long all_work = 0;
  for (int i = 0; i < 16; ++i) all_work += sums[i];
  const int most = (int)max((5 * all_work + 4LL * n - 1) / (4LL * n), 8LL);  // of a part
  const int parts = j < n ? min(max((x + most - 1) / most, 1), kMaxParts) : 0;
  int cut = j < n && (long long)x * n > all_work ? block[kScheduleHead + 3 * n + schedule_jobs(n) + j] : 0;
  const float jobs_here = wave_sum((float)parts), cut_here = wave_sum(cut ? 1.f : 0.f);
  if (lane == 0) counts[wave] = (int)jobs_here, cuts_here[wave] = (int)cut_here;
  keys[j] = make_int4(x << 10 | j, 0, 0, cut);
  __syncthreads();
  int jobs = 0, cut_tiles = 0;
  for (int i = 0; i < 16; ++i) jobs += counts[i], cut_tiles += cuts_here[i];
  if (cut_tiles > n / 4) {  // the most work only
    int more = 0;
    if (cut)
      for (int i = 0; i < n; ++i) more += keys[i].w && keys[i].x > (x << 10 | j);
    if (more >= n / 4) cut = 0;
    cut_tiles = n / 4;
    __syncthreads();
  }
  const int whole = x << 10 | j, part = parts ? ((x + parts - 1) / parts << 10 | j) << 3 | (parts - 1) : 0;
  // the rows of a cut tile before the cut and from it on; the later piece of equal ones begins first
  const int before = cut ? ((cut >> 7) & 1023) << 10 | j : whole, from = cut ? cut >> 17 << 10 | j : -1;
  keys[j] = make_int4(whole, part, before, from);
  __syncthreads();
  if (slice == 0 && j == 0) block[0] = jobs, block[1] = n + cut_tiles;
  const int per = kMostTiles / slices, tile = slice * per + j;
  if (j >= per || tile >= n) return;
  const int4 here = keys[tile];
  int rank = 0, first = 0, rank_before = here.w >= here.z, rank_from = 0;
  for (int i = 0; i < n; ++i) {
    const int4 k = keys[i];
    rank += k.x > here.x;
    first += k.y > here.y ? (k.y & 7) + 1 : 0;
    rank_before += (k.z > here.z) + (k.w > here.z);
    if (here.w >= 0) rank_from += (k.z > here.w) + (k.w > here.w);
  }
  rank_before -= here.w > here.z;  // counted above
  const int at = here.w >= 0 ? block[kScheduleHead + 3 * n + schedule_jobs(n) + tile] & 127 : 0;
  int* pieces = block + kScheduleHead + 4 * n + schedule_jobs(n);
  pieces[rank_before] = tile | (at ? at - 1 : kRowTile - 1) << 17;
  if (at) pieces[rank_from] = tile | at << 10 | (kRowTile - 1) << 17;
  block[kScheduleHead + n + rank] = tile;
  const int of = (here.y & 7) + 1;
  block[kScheduleHead + 2 * n + tile] = first | of << 24;
  int* jobs_at = block + kScheduleHead + 3 * n + first;
  for (int p = 0; p < of; ++p) jobs_at[p] = tile | p << 20 | (of - 1) << 23;
}

// Shape of the launch: rows per workgroup, tiles and splits.
int plan(const musc_masked_attention& c, Args& a, int& waves) {
  a.c = c;
  a.group = c.heads / c.kv_heads;
  const long long rows = (long long)c.q_len * a.group;
  if (rows > 0x7fffff00LL || c.k_len > 0x7fffff00) return MUSC_ERR_UNSUPPORTED;
  a.rows = (int)rows;
  waves = rows <= 32 ? 1 : 4;
  const int tile = waves == 1 || c.dtype == MUSC_DTYPE_F32 ? 32 : 64;
  a.row_tiles = (int)((rows + 32 * waves - 1) / (32 * waves));
  a.key_tiles = (c.k_len + tile - 1) / tile;
  a.summaries = (c.k_len + kSummaryKeys - 1) / kSummaryKeys;
  const long long heads = (long long)c.batch * c.kv_heads, whole = heads * a.row_tiles;
  // workgroups that the card holds at a time
  a.slots = waves == 1 ? 1024 : c.dtype != MUSC_DTYPE_F32 && c.d <= 64 ? 768 : 512;
  a.splits = 1, a.jobs = a.row_tiles, a.in_parts = 0, a.in_pieces = 0, a.teams = 1;
  // Few rows over up to 2048 keys (1024 of wide heads): the waves of one workgroup share them and
  // join in LDS, without a second launch.  One row, 1369 keys, 16 heads of 64: 17.1 us in
  // workgroups of one wave and a join, 12.9 us so, host time included.
  const int teams = teams_of((c.d <= 64 ? 64 : 128) * (c.dtype == MUSC_DTYPE_F32 ? 4 : 2));
  if (waves == 1 && a.key_tiles <= kTeamTiles * teams) a.teams = teams;
  if (a.teams > 1) {
  } else if (waves > 1 && c.schedule) {
    // No splits: pieces and parts even out documents of different lengths, and one document alone, or equal
    // ones, gain nothing (1370 tokens, fp16, heads of 64: 27 us for 4, 8 or 16 heads; in splits 25, 36 and 50.
    // fp32, 4 heads: 115, in splits 45; 600 tokens, heads of 128: 102, in splits 38 to 42).
    // Where all row tiles begin at once the longest ends last.  With an order of tokens their lengths
    // differ most: long ones go in parts, if long enough to pay for a join (fp16, 8 heads of 64: three
    // causal documents of 4000 tokens in all 45 us, in pieces 58; of 1000 20 us either way).  So do those
    // of fp32 with narrow heads, whose tiles take longest (4 packed images 227 us, in pieces 256; four
    // documents of 1000 tokens in all 47, 60; three 69, 54).
    a.in_parts = whole < a.slots && (c.q_order ? c.dtype == MUSC_DTYPE_F32 || c.k_len >= 2048 : c.dtype == MUSC_DTYPE_F32 && c.d <= 64);
    if (a.in_parts) a.jobs = (int)schedule_jobs(a.row_tiles);
    // Without an order the longest tiles are those that end one document and begin the next: cut there
    // (fp16, 16 heads of 64: 12 packed images 99 us whole, 87 in pieces; three documents of 1500 tokens in
    // all 49, 29, of 2500 with a bias 66 in parts, 46 in pieces).  Few rounds only: listed but empty
    // pieces cost a little, and short tiles fill up behind long ones.
    a.in_pieces = !a.in_parts && !c.q_order && whole < 4LL * a.slots;
    if (a.in_pieces) a.jobs = (int)schedule_pieces(a.row_tiles);
  } else if (whole < (waves == 1 ? 1024 : 256)) {
    // few rows: their keys in splits of at least one tile (4 where four waves share the tiles)
    long long splits = ((waves == 1 ? 2048 : 512) + whole - 1) / whole;
    const int least = waves == 1 ? 1 : 4;
    if (splits > a.key_tiles / least) splits = a.key_tiles / least;
    if (splits > kMaxSplits) splits = kMaxSplits;
    a.splits = splits < 1 ? 1 : (int)splits;
  }
  a.units = heads * a.jobs * a.splits;
  // Heads that an XCD (32 CUs, 2 or 3 workgroups each) works on together: enough for two rounds of
  // workgroups, so that short work fills the gaps of long work, and no more, as they share its L2.
  // 0: the heads do not divide over the XCDs.
  a.heads_at_once = 0;
  if (heads % kXcds == 0) {
    const long long enough = (128 + a.row_tiles - 1) / a.row_tiles, per_xcd = heads / kXcds;
    a.heads_at_once = (int)(enough < per_xcd ? enough : per_xcd);
  }
  // a grid dimension holds fewer than 2^32 threads, 256 or (teams) up to 512 a workgroup
  if (a.units >= (0x100000000LL >> (a.teams > 1 ? 9 : 8))) return MUSC_ERR_UNSUPPORTED;
  return MUSC_OK;
}

// Rows that write parts: of every split, or of every job.
size_t part_rows(const Args& a) {
  const size_t heads = (size_t)a.c.batch * a.c.kv_heads;
  if (a.in_parts) return heads * a.jobs * kRowTile;
  return a.splits == 1 ? 0 : heads * a.rows * a.splits;
}
size_t part_bytes(const Args& a) {
  const size_t rows = part_rows(a);
  return rows ? align_up(rows * 2 * sizeof(float), 256) + rows * a.c.d * sizeof(float) : 0;
}

// 16-byte vectors from every row of a tensor
inline bool aligned(const void* p, long long sb, long long st, long long sh, int per) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb >= 0 && st >= 0 && sh >= 0 && (sb | st | sh) % per == 0;
}

int check(const musc_masked_attention* c) {
  if (!c || !c->q || !c->k || !c->v || !c->out) return MUSC_ERR_INVALID_ARG;
  if (c->dtype != MUSC_DTYPE_F32 && c->dtype != MUSC_DTYPE_F16 && c->dtype != MUSC_DTYPE_BF16) return MUSC_ERR_INVALID_ARG;
  if (c->batch < 1 || c->q_len < 1 || c->k_len < 1 || c->heads < 1 || c->kv_heads < 1 || c->heads % c->kv_heads)
    return MUSC_ERR_INVALID_ARG;
  // scores, slopes and the cap are taken relative to one another
  const float least = 0x1p-60f, most = 0x1p60f;
  if (!(c->cap >= 0.f) || (c->cap > 0.f && !(c->cap >= least && c->cap <= most))) return MUSC_ERR_INVALID_ARG;
  if (!(fabsf(c->scale) <= most) || (c->scale != 0.f && fabsf(c->scale) < least)) return MUSC_ERR_INVALID_ARG;
  const int per = c->dtype == MUSC_DTYPE_F32 ? 4 : 8, size = 16 / per;
  if (c->d < 1 || c->d > 128 || c->d % per) return MUSC_ERR_UNSUPPORTED;
  if (!aligned(c->q, c->q_sb, c->q_st, c->q_sh, per) || !aligned(c->k, c->k_sb, c->k_st, c->k_sh, per) ||
      !aligned(c->v, c->v_sb, c->v_st, c->v_sh, per) || !aligned(c->out, c->o_sb, c->o_st, c->o_sh, per))
    return MUSC_ERR_INVALID_ARG;
  if (c->k_st > kNowhere || c->v_st > kNowhere || (63 * c->k_st + c->d) * size > kNowhere - 16 ||
      (63 * c->v_st + c->d) * size > kNowhere - 16)
    return MUSC_ERR_UNSUPPORTED;
  // documents on both sides and the keys' summary, or none; orders and positions likewise
  if (!c->q_documents != !c->k_documents || !c->k_documents != !c->k_summary) return MUSC_ERR_INVALID_ARG;
  if (!c->q_order != !c->k_order || (c->q_order && !c->q_documents)) return MUSC_ERR_INVALID_ARG;
  if (c->axes < 0 || c->axes > kMaxAxes) return MUSC_ERR_UNSUPPORTED;
  if (c->axes && (!c->q_positions || !c->k_positions || !c->slopes)) return MUSC_ERR_INVALID_ARG;
  const uintptr_t words = reinterpret_cast<uintptr_t>(c->q_documents) | reinterpret_cast<uintptr_t>(c->k_documents) |
                          reinterpret_cast<uintptr_t>(c->q_order) | reinterpret_cast<uintptr_t>(c->k_order) |
                          reinterpret_cast<uintptr_t>(c->q_positions) | reinterpret_cast<uintptr_t>(c->k_positions) |
                          reinterpret_cast<uintptr_t>(c->slopes) | reinterpret_cast<uintptr_t>(c->schedule);
  if ((words & 3) || (reinterpret_cast<uintptr_t>(c->k_summary) & 15)) return MUSC_ERR_INVALID_ARG;
  if ((c->q_tokens_sb | c->k_tokens_sb | c->q_positions_sb | c->k_positions_sb | c->k_summary_sb |
       c->schedule_sb) < 0)
    return MUSC_ERR_INVALID_ARG;
  return MUSC_OK;
}

}  // namespace mattn
}  // namespace musc

using namespace musc;

extern "C" int musc_token_summary(const int* documents, const int* order, int batch, int t, int* summary,
                                  hipStream_t stream) {
  if (!documents || !summary || batch < 0 || t < 0) return MUSC_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(documents) | reinterpret_cast<uintptr_t>(order)) & 3) ||
      (reinterpret_cast<uintptr_t>(summary) & 15))
    return MUSC_ERR_INVALID_ARG;
  if (batch == 0 || t == 0) return MUSC_OK;
  const int groups = (int)(((long long)t + mattn::kSummaryKeys - 1) / mattn::kSummaryKeys);
  const long long blocks = ((long long)batch * groups * mattn::kSummaryKeys + 255) / 256;
  if (blocks >= (0x100000000LL >> 8)) return MUSC_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(mattn::token_summary_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, documents, order, batch,
                     t, groups, reinterpret_cast<int4*>(summary));
  return check_launch();
}

extern "C" int musc_token_schedule(const int* documents, const int* order, const int* summary, int batch, int t,
                                   int* schedule, hipStream_t stream) {
  if (!documents || !summary || !schedule || batch < 0 || t < 0) return MUSC_ERR_INVALID_ARG;
  if (((reinterpret_cast<uintptr_t>(documents) | reinterpret_cast<uintptr_t>(order) |
        reinterpret_cast<uintptr_t>(schedule)) & 3) || (reinterpret_cast<uintptr_t>(summary) & 15))
    return MUSC_ERR_INVALID_ARG;
  if (t > MUSC_SCHEDULE_MAX_TOKENS) return MUSC_ERR_UNSUPPORTED;
  if (batch == 0 || t == 0) return MUSC_OK;
  mattn::Schedule s{};
  s.batch = batch, s.t = t, s.groups = (t + mattn::kSummaryKeys - 1) / mattn::kSummaryKeys;
  for (int w = 0; w < 4; ++w) {
    s.tiles[w] = (t + (mattn::kRowTile >> w) - 1) / (mattn::kRowTile >> w);
    s.first[w + 1] = s.first[w] + (long long)batch * s.tiles[w];
    if (w < 3) s.at[w + 1] = s.at[w] + batch * mattn::schedule_block(s.tiles[w]);
  }
  if (s.first[4] >= (0x100000000LL >> 10)) return MUSC_ERR_UNSUPPORTED;
  hipLaunchKernelGGL(mattn::row_work_kernel, dim3((unsigned)s.first[4]), dim3(kWave), 0, stream, documents, order,
                     reinterpret_cast<const int4*>(summary), s, schedule);
  const int slices = s.tiles[3] > 256 ? 4 : 1;  // 1370 tokens 8 us, 4096 14; 9465 30, 16384 48 (one workgroup: 151)
  hipLaunchKernelGGL(mattn::row_order_kernel, dim3((unsigned)(batch * 4 * slices)), dim3(1024), 0, stream, s, slices,
                     schedule);
  return check_launch();
}

extern "C" int musc_masked_attention_workspace_bytes(const musc_masked_attention* c, size_t* out) {
  if (!out) return MUSC_ERR_INVALID_ARG;
  if (const int rc = mattn::check(c)) return rc;
  mattn::Args a{};
  int waves;
  if (const int rc = mattn::plan(*c, a, waves)) return rc;
  *out = mattn::part_bytes(a);
  return MUSC_OK;
}

extern "C" int musc_masked_attention_fwd(const musc_masked_attention* c, void* workspace, size_t workspace_bytes,
                                         hipStream_t stream) {
  if (const int rc = mattn::check(c)) return rc;
  mattn::Args a{};
  int waves;
  if (const int rc = mattn::plan(*c, a, waves)) return rc;
  const size_t need = mattn::part_bytes(a);
  if (need) {
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16) return MUSC_ERR_WORKSPACE;
    a.part_ml = static_cast<float*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                        align_up(mattn::part_rows(a) * 2 * sizeof(float), 256));
  }
  if (c->dtype == MUSC_DTYPE_F32) mattn::launch_f32(a, waves, stream);
  else if (c->dtype == MUSC_DTYPE_F16) mattn::launch_f16(a, waves, stream);
  else mattn::launch_bf16(a, waves, stream);
  return check_launch();
}
