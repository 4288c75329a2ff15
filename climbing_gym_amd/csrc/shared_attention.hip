// Decode attention for rows in groups that share the first part of their history (the completions of one prompt): the
// shared positions are read once for all rows of a group, each row's own positions once, and the partial softmaxes joined.
//
// Cache addressing is that of attention.hip: element (slot, pos, head, d) at slot*c0 + pos*c1 + head*c2 + d, the e4m3 scale
// of (slot, pos, head) at that offset divided by D; with a block table c0 is the page stride and pos the in-page index.
#include "lfm2_common.h"
#include <type_traits>

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr int kStep = 32;                 // history tokens that meet 16 queries at a time
constexpr int kShareTile = 4 * kStep;     // tokens a workgroup stages at a time of a part that a group shares
// Chunks are multiples of this: those of a workgroup, those of a wave (128 for both: 16 rows of 900 tokens 12.4 us instead of
// 11.2, six layers of 16 x 16 rows 318 instead of 308; 55 paged rows of 128 dims 36.7 instead of 38.4).
constexpr int kGrain = 128, kWaveGrain = 64;
constexpr int kMaxRows = 4096;            // rows and groups the work list holds
constexpr int kSplitSlots = 2048;         // partial results beyond one per row and part, for the shared parts and for the others
constexpr int kQueryTile = 64;            // queries of an item that a group shares: its (row, head) pairs of one KV head
constexpr int kQueryBlock = 16;           // queries of the other items
constexpr int kTurn = 256;                // workgroups, one per CU
constexpr int kSharedBlocks = 2 * kTurn, kOtherBlocks = 3 * kTurn;
constexpr int kSharedItems = 512;      // items the shared parts are cut into, if their length allows ...
// ... and the others, as items of a wave and of a workgroup (256 rows with own parts of 2000 tokens, e4m3: 112 us with 2048
// long items, 122 with 4096; six layers of 16 x 16 rows with up to 900: 282 us with 4096 short ones, 300 with 2048).
constexpr int kShortItems = 4096, kLongItems = 2048;
// Parts of up to this many tokens are waves' items, longer ones workgroups'.  A workgroup's waves read four tiles in a row, which
// the memory likes, and pay for their join; waves' items fill the chip more evenly.  With 2048 instead of 1024: 4 x 16 rows with
// own parts of 1 to 4000 tokens 57 us instead of 62 (e4m3: 47 instead of 53), 256 rows of 2000 181 instead of 177 (117, 113).
// Waves' items alone: one row of 60000 54 us instead of 35, 64 rows of 6000 135 instead of 122.
constexpr int kWaveTokens = 2048;

// ---- the work list (int32), built once per decode step and used by every attention layer
//   header: what the list was built for, number of records of each of the three kinds of item
//   one record per row: first partial result, shared chunks, own chunks, length (0: sits out)
//   one record per item, kind after kind: first row, rows, query tile, place of the partial result among the row's, first
//   token, end token, slot or table row that holds them, whose tokens they are (kOwn, kShared, kCut)
// A group with more queries than a block has its shared part cut into "shared" items, of a workgroup and up to 64 queries.
// Everything else (rows' own parts, the shared parts of smaller groups) becomes items of one block of queries: a workgroup's
// ("long"), or a wave's ("short") where the part has at most kWaveTokens tokens.
enum { kHShared, kHLong, kHShort, kHRows, kHCapacity, kHQueryHeads, kHKvHeads, kHDim, kHeader = 16 };
constexpr int kRowInts = 4, kRecordInts = 8;
// A row that ends inside its group's prefix takes no part in the shared items: it would meet the tokens behind its end with
// weight 0, and 0 times an infinity there is not 0.  It reads its piece of the prefix by itself (kCut).
enum { kOwn, kShared, kCut };

struct SlotBounds { int64_t slots, records; };
// Upper bounds of the partial results and of the items of a batch, from what the host knows.  A row has at most
// ceil(capacity / kWaveGrain) shared and as many own chunks; a chunk size is at least 1 / kSplitSlots of the tokens it cuts (with
// multiplicity, the shared ones counted once per row), so the shared parts and the others make at most kSplitSlots chunks each
// plus one per part, and a row has two parts.  An item covers at least one row's queries, or a tile of them.
SlotBounds slot_bounds(int64_t B, int64_t capacity, int G) {
  const int64_t per_row = (capacity + kWaveGrain - 1) / kWaveGrain;
  const int64_t half = B * per_row < B + kSplitSlots ? B * per_row : B + kSplitSlots;
  return SlotBounds{2 * half, 2 * half * ((G + kQueryBlock - 1) / kQueryBlock)};
}
int64_t schedule_ints(int64_t B, int64_t capacity, int G) {
  return kHeader + kRowInts * B + kRecordInts * slot_bounds(B, capacity, G).records;
}

struct ScheduleArgs {
  int32_t* schedule;
  const int32_t *positions, *slot_ids, *starts, *prefix_slots, *prefix_lengths;
  const uint8_t* active;
  int64_t capacity;
  int B, groups, QH, KH, G, D;
};

__device__ __forceinline__ int round_up(int v, int step) { return (v + step - 1) / step * step; }

// ceil(x / y) of positive numbers (x below 2^26) through a float reciprocal and an exact correction by one: an integer
// division is forty instructions, and the work list's kernel has many.
__device__ __forceinline__ int divide_up(int x, int y, float inverse) {
  const int n = x + y - 1;
  const int q = (int)((float)n * inverse), rest = n - q * y;
  return q + (rest >= y ? 1 : rest < 0 ? -1 : 0);
}
__device__ __forceinline__ int divide_up(int x, int y) { return divide_up(x, y, __builtin_amdgcn_rcpf((float)y)); }
// How parts are cut: into pieces of at most `units` times kWaveGrain tokens.
struct Cut {
  int units;
  float inverse;
  static __device__ __forceinline__ Cut of(int size) {
    return Cut{size / kWaveGrain, __builtin_amdgcn_rcpf((float)(size / kWaveGrain))};
  }
  // field by field: a choice between objects would put them into memory
  static __device__ __forceinline__ Cut choose(bool first, const Cut a, const Cut b) {
    return Cut{first ? a.units : b.units, first ? a.inverse : b.inverse};
  }
  __device__ __forceinline__ int pieces(int tokens) const { return divide_up((tokens + kWaveGrain - 1) / kWaveGrain, units, inverse); }
};

// Four sums, and four exclusive prefix sums with their totals, over 1024 threads.
__device__ __forceinline__ f32x4 sum4_1024(f32x4 v, f32x4* scratch) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = wave_sum(v[i]);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  f32x4 t = scratch[0];
#pragma unroll
  for (int w = 1; w < 16; ++w) t += scratch[w];
  return t;
}
__device__ __forceinline__ i32x4 scan4_1024(const i32x4 v, i32x4* scratch, i32x4* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  i32x4 x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int up = __shfl_up(x[i], o, 64);
      if (lane >= o) x[i] += up;
    }
  }
  if (lane == 63) scratch[wave] = x;
  __syncthreads();
  i32x4 before = {0, 0, 0, 0}, all = {0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const i32x4 t = scratch[w];
    if (w < wave) before += t;
    all += t;
  }
  *total = all;
  return before + x - v;
}

// One workgroup.  A thread has PER rows and PER groups (one each up to 1024 of them).  Its time is that of its dependent
// rounds: everything is read from memory at the start, at once, and the sums and places of all kinds go through two joins.
// 8 us up to 1024 rows, 16 to 22 for 2048 to 4096 (4096 groups of one row: 37).
template <int PER>
__global__ void __launch_bounds__(1024) shared_schedule_kernel(ScheduleArgs a) {
  constexpr int MOST = 1024 * PER;
  __shared__ int starts[MOST + 1], extent[MOST], source[MOST], prefix[MOST];
  __shared__ f32x4 fscratch[16];
  __shared__ i32x4 scratch[16];
  const int tid = threadIdx.x, G = a.G, capacity = (int)a.capacity;
  int length[PER], slot_of[PER], group[PER], shared[PER];   // shared: positions a row has in common with its group, 0: none
  bool cut[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    length[i] = slot_of[i] = 0;
    if (b < a.B) {
      const int position = a.positions[b];
      slot_of[i] = a.slot_ids ? a.slot_ids[b] : b;
      const bool on = (!a.active || a.active[b]) && slot_of[i] >= 0 && position >= 0;
      length[i] = !on ? 0 : position < capacity ? position + 1 : capacity;
    }
    if (b < a.groups) {
      const int s = a.starts[b], p = a.prefix_lengths[b];
      starts[b] = s < 0 ? 0 : s > a.B ? a.B : s;
      prefix[b] = p < 0 ? 0 : p > capacity ? capacity : p;
      source[b] = a.prefix_slots[b];
      extent[b] = 0;
    }
  }
  if (tid == 0) {
    const int s = a.starts[a.groups];
    starts[a.groups] = s < 0 ? 0 : s > a.B ? a.B : s;
  }
  __syncthreads();
  // bounds out of order would give a row to several groups: such a list is marked as nobody's (its users return NaN)
  int disorder = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) disorder |= tid * PER + i < a.groups && starts[tid * PER + i] > starts[tid * PER + i + 1];
  if (__syncthreads_or(disorder)) {
    if (tid == 0) a.schedule[kHRows] = -1;
    return;
  }
  // a row's group: the last one that starts at or before it
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    group[i] = -1;
    shared[i] = 0;
    cut[i] = false;
    if (b >= a.B) continue;
    int lo = 0, hi = a.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= b) lo = mid; else hi = mid;
    }
    if (starts[lo] <= b && b < starts[lo + 1] && source[lo] >= 0) {
      cut[i] = length[i] < prefix[lo];
      if (cut[i]) {
        slot_of[i] = source[lo];
      } else {
        group[i] = lo;
        shared[i] = prefix[lo];
        extent[lo] = prefix[lo];   // the same value from every row of the group
      }
    }
  }
  __syncthreads();
  // chunk sizes: enough items to fill the chip, no more partial results than the workspace holds
  auto queries = [&](int g) { return (starts[g + 1] - starts[g]) * G; };
  auto wide = [&](int g) { return queries(g) > kQueryBlock; };
  const int own_tiles = (G + kQueryBlock - 1) / kQueryBlock;
  float wide_tokens = 0.f, other_tokens = 0.f, wide_work = 0.f, other_work = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    if (b >= a.B) continue;
    if (group[i] >= 0) (wide(group[i]) ? wide_tokens : other_tokens) += (float)extent[group[i]];
    if (length[i] > shared[i]) {
      other_tokens += (float)(length[i] - shared[i]);
      other_work += (float)(length[i] - shared[i]) * (float)own_tiles;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int g = tid * PER + i;
    if (g >= a.groups) continue;
    if (wide(g)) wide_work += (float)extent[g] * (float)((queries(g) + kQueryTile - 1) / kQueryTile);
    else other_work += (float)extent[g];
  }
  const f32x4 sums = sum4_1024(f32x4{wide_tokens, other_tokens, wide_work, other_work}, fscratch);
  auto chunk_of = [&](float tokens, float work, int items, int grain) {
    // a little more than the quotient: the sums are rounded.  (6e8 is above 2^40 tokens over kSplitSlots, and twice it an int.)
    const float need = fmaxf(tokens / (float)kSplitSlots, work * (float)a.KH / (float)items);
    return round_up((int)fminf(need * 1.0001f, 6.0e8f) + 1, grain);
  };
  // The shared parts' chunk: of sixteen sizes up to about twice the smallest that will do, the one that is done first.  One
  // wave tries one size.  Two workgroups on a CU do twice as many tokens in 1.4 of the time, and cost 256 tokens' time more
  // than one (they start one after the other, and their partial results are written and joined): 16 x 16 rows, e4m3, 4000
  // shared tokens as 512 items of 1024 take 35 us, as 256 of 2048 43; 4 x 16 rows, 2000 tokens, 512 of 128 19, 256 of 256 15;
  // about 1000 tokens for each CU are done in the same time either way.
  const int smallest = chunk_of(sums[0], sums[2], kSharedItems, kGrain), step = round_up(smallest / 16 + 1, kGrain);
  {
    const int wave = tid >> 6, chunk = smallest + wave * step;
    const Cut cut = Cut::of(chunk);
    int items = 0;
    for (int g = tid & 63; g < a.groups; g += 64)
      if (wide(g)) items += cut.pieces(extent[g]) * ((queries(g) + kQueryTile - 1) / kQueryTile);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) items += __shfl_xor(items, o, 64);
    if ((tid & 63) == 0) scratch[wave][0] = __builtin_bit_cast(int, items * a.KH <= kTurn ? (float)chunk : (float)((items * a.KH + kSharedBlocks - 1) / kSharedBlocks) * (1.4f * (float)chunk + 256.f));
    __syncthreads();
  }
  int wide_chunk = smallest, least = scratch[0][0];   // positive floats are in order as integers too
#pragma unroll
  for (int c = 1; c < 16; ++c) {
    const int cost = scratch[c][0];
    if (cost < least) { least = cost; wide_chunk = smallest + c * step; }
  }
  __syncthreads();
  const Cut wide_cut = Cut::of(wide_chunk), long_cut = Cut::of(chunk_of(sums[1], sums[3], kLongItems, kGrain)),
            short_cut = Cut::of(chunk_of(sums[1], sums[3], kShortItems, kWaveGrain));
  // a part's chunks, and its records by kind (0 shared, 1 long, 2 short)
  struct Part {
    int chunk, chunks, tiles, records, kind;
    // pieces of the same size: the longest decides when the launch is done
    __device__ __forceinline__ void split(int tokens, const Cut cut, int grain) {
      const int units = (tokens + kWaveGrain - 1) / kWaveGrain, most = max(cut.pieces(tokens), 1);
      const int each = round_up(divide_up(units, most), grain / kWaveGrain);
      chunk = each * kWaveGrain;
      chunks = tokens > 0 ? divide_up(units, each) : 0;
    }
  };
  auto shared_part = [&](int g) {
    Part p;
    p.kind = wide(g) ? 0 : extent[g] > kWaveTokens ? 1 : 2;
    p.split(extent[g], Cut::choose(p.kind == 0, wide_cut, Cut::choose(p.kind == 1, long_cut, short_cut)), p.kind == 2 ? kWaveGrain : kGrain);
    p.tiles = wide(g) ? (queries(g) + kQueryTile - 1) / kQueryTile : 1;
    p.records = p.chunks * p.tiles;
    return p;
  };
  auto own_part = [&](int tokens) {
    Part p;
    p.kind = tokens > kWaveTokens ? 1 : 2;
    p.split(tokens, Cut::choose(p.kind == 1, long_cut, short_cut), p.kind == 2 ? kWaveGrain : kGrain);
    p.tiles = own_tiles;
    p.records = p.chunks * own_tiles;
    return p;
  };
  // places: partial results of every row, then the records, kind after kind
  int slots = 0, shared_records = 0, long_records = 0, short_records = 0;
  int np[PER], ns[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    np[i] = ns[i] = 0;
    if (b < a.B) {
      if (group[i] >= 0) np[i] = shared_part(group[i]).chunks;
      const Part own = own_part(length[i] - shared[i]);
      ns[i] = own.chunks;
      slots += np[i] + ns[i];
      long_records += own.kind == 1 ? own.records : 0;
      short_records += own.kind == 2 ? own.records : 0;
    }
    if (b < a.groups) {   // the same numbers once more, for groups
      const Part part = shared_part(b);
      shared_records += part.kind == 0 ? part.records : 0;
      long_records += part.kind == 1 ? part.records : 0;
      short_records += part.kind == 2 ? part.records : 0;
    }
  }
  i32x4 totals;
  const i32x4 first = scan4_1024(i32x4{shared_records, long_records, short_records, slots}, scratch, &totals);
  int shared_at = first[0], long_at = totals[0] + first[1], short_at = totals[0] + totals[1] + first[2], slot = first[3];
  int32_t* const records = a.schedule + kHeader + kRowInts * a.B;
  // writes a part's records from `place` on
  auto put = [&](const Part part, int place, int row, int rows, int offset, int t0, int end, int source, int whose) {
    i32x4* r = reinterpret_cast<i32x4*>(records) + 2 * (int64_t)place;
    for (int c = 0; c < part.chunks; ++c, t0 += part.chunk)
      for (int qt = 0; qt < part.tiles; ++qt, r += 2) {
        r[0] = i32x4{row, rows, qt, offset + c};
        r[1] = i32x4{t0, min(t0 + part.chunk, end), source, whose};
      }
  };
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    if (b < a.B) {
      *reinterpret_cast<i32x4*>(a.schedule + kHeader + kRowInts * b) = i32x4{slot, np[i], ns[i], length[i]};
      slot += np[i] + ns[i];
      const Part part = own_part(length[i] - shared[i]);
      put(part, part.kind == 1 ? long_at : short_at, b, 1, np[i], shared[i], length[i], slot_of[i], cut[i] ? kCut : kOwn);
      long_at += part.kind == 1 ? part.records : 0;
      short_at += part.kind == 2 ? part.records : 0;
    }
    if (b < a.groups) {
      const Part part = shared_part(b);
      put(part, part.kind == 0 ? shared_at : part.kind == 1 ? long_at : short_at, starts[b], starts[b + 1] - starts[b], 0, 0, extent[b],
          source[b], kShared);
      shared_at += part.kind == 0 ? part.records : 0;
      long_at += part.kind == 1 ? part.records : 0;
      short_at += part.kind == 2 ? part.records : 0;
    }
  }
  if (tid == 0) {
    a.schedule[kHShared] = totals[0];
    a.schedule[kHLong] = totals[1];
    a.schedule[kHShort] = totals[2];
    a.schedule[kHRows] = a.B;
    a.schedule[kHCapacity] = capacity;
    a.schedule[kHQueryHeads] = a.QH;
    a.schedule[kHKvHeads] = a.KH;
    a.schedule[kHDim] = a.D;
  }
}

// ===================================================================================== attention
template <typename T> struct HalfMfma;
template <> struct HalfMfma<__bf16> {
  typedef bf16x8 vec8;
  static __device__ __forceinline__ f32x4 run(vec8 a, vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct HalfMfma<_Float16> {
  typedef f16x8 vec8;
  static __device__ __forceinline__ f32x4 run(vec8 a, vec8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Eight e4m3 codes (two dwords) to eight values of T: exact in either type.
template <typename T> __device__ __forceinline__ typename HalfMfma<T>::vec8 widen8(int lo, int hi);
template <> __device__ __forceinline__ bf16x8 widen8<__bf16>(int lo, int hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <> __device__ __forceinline__ f16x8 widen8<_Float16>(int lo, int hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Lanes of a wave exchange values through LDS: the hardware keeps a wave's LDS accesses in order, and this keeps the
// compiler from moving or reusing them across the exchange.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

struct SharedArgs {
  void* out;
  const void *q, *kc, *vc;
  const float *ks, *vs;
  const int32_t *schedule, *table;
  float *acc, *m, *l;          // partial results: [slot][query head][D], [slot][query head] twice
  int64_t c0, c1, c2, max_blocks, pools, sources;   // pools: slots or pages; sources: slots or table rows
  int page, page_shift, B, QH, KH, G, capacity, shared_blocks, other_blocks;
  float scale_log2e;
};
__device__ __forceinline__ bool list_fits(const SharedArgs& a, int D) {
  const int32_t* s = a.schedule;
  return s[kHRows] == a.B && s[kHCapacity] == a.capacity && s[kHQueryHeads] == a.QH && s[kHKvHeads] == a.KH && s[kHDim] == D;
}

// How 16 queries meet 32 tokens (lane % 16 = r is the lane's query throughout, grp = lane / 16):
//   S^T  = K . Q^T   (A = 16 tokens x 32 dims, B = 32 dims x 16 queries): the lane gets tokens 4 grp + i of its query;
//   O^T += V^T . P^T (A = V^T through the transposing read of the row-major LDS tile, B = P straight from the S^T registers),
// so softmax statistics never cross queries and P needs no relayout.  The running maximum is raised only when a score
// exceeds it by more than 8 (powers of two), so most tiles need no rescaling: p <= 2^8 fits every type used here and the
// reference point cancels in the end.
// The second product takes 16-bit operands.  A 16-bit history's P goes in as two of them, the rounded value and the rounded
// rest (2^-16 relative in bf16: one rounding alone would be as large as the output's own).  An e4m3 history's goes in as one
// fp16 value (2^-11, and 2^-25 of the largest weight below fp16's normal range: less than a bf16 output's own rounding, as much
// as an fp16 one's), with the scale of its V row: the weight is w = 2^{s + log2 vs - m}, m a running maximum of s + log2 vs,
// so it stays in fp16's range whatever the scales are, and the softmax sum takes w / vs.
template <typename T, bool FP8, int D> struct Shape {
  typedef std::conditional_t<FP8, _Float16, T> P;   // type of P and V: fp16 holds e4m3 exactly, and three more bits of P than bf16
  typedef typename HalfMfma<T>::vec8 kvec;
  typedef typename HalfMfma<P>::vec8 pvec;
  static constexpr int ES = FP8 ? 1 : 2, RB = D * ES;   // bytes per element and per row of the history
  static constexpr int KK = D / 32;                     // products per 16 x 16 scores
  static constexpr int KC = D / 8;                      // 16-byte pieces of a row of 16-bit values in LDS
  static constexpr int ROW16 = RB / 16;                 // 16-byte pieces of a row of the history
};

// Scales of a tile's tokens in LDS: of K with the score scale and log2 e, log2 of V's and its inverse.
struct Scales {
  float *k, *log_v, *inverse_v;
  __device__ __forceinline__ Scales operator+(int t) const { return Scales{k + t, log_v + t, inverse_v + t}; }
  __device__ __forceinline__ void set_v(int t, float vs) const {
    // a scale of 0 (its row is all zeros) takes part in the softmax sum and adds nothing: 2^-80 does the same
    vs = vs < 8.2718061e-25f ? 8.2718061e-25f : vs;
    log_v[t] = __builtin_amdgcn_logf(vs);
    inverse_v[t] = __builtin_amdgcn_rcpf(vs);
  }
};

template <typename T, bool FP8, int D> struct QueryBlock {
  typedef Shape<T, FP8, D> S;
  typename S::kvec q[S::KK];
  f32x4 o[D / 16];
  float m, l;
  int place;   // row of the partial results, -1: nowhere

  __device__ __forceinline__ void start(const SharedArgs& a, const i32x4 r0, int whose, int h, int q0) {
    const int lane = threadIdx.x & 63, r = lane & 15, grp = lane >> 4;
    const int row0 = r0[0], total = r0[1] * a.G, qi = min(q0 + r, total - 1);
    const int b = row0 + qi / a.G, head = h * a.G + qi % a.G;
    const T* src = (const T*)a.q + ((int64_t)b * a.QH + head) * D;
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk) q[kk] = *reinterpret_cast<const typename S::kvec*>(src + 32 * kk + 8 * grp);
    const i32x4 record = *reinterpret_cast<const i32x4*>(a.schedule + kHeader + kRowInts * b);
    // a row that sits out, or ends inside the prefix, computes something that is never stored
    const bool mine = q0 + r < total && record[3] > 0 && (whose != kShared || r0[3] < record[1]);
    place = mine ? (record[0] + r0[3]) * a.QH + head : -1;
    m = -kInf;
    l = 0.f;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) o[dd] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  __device__ __forceinline__ void raise(float top) {   // a new maximum of the query, the same in its four lanes
    const float mnew = fmaxf(m, top);
    const float alpha = mnew == -kInf ? 1.f : __builtin_amdgcn_exp2f(m - mnew);
    m = mnew;
    l *= alpha;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dd][i] *= alpha;
  }
  // A wave's results to LDS, lane by lane, and another wave's joined to one's own.
  static constexpr int kShare = 64 * (D / 4 + 2);   // floats
  __device__ __forceinline__ void hand_over(float* to) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int i = 0; i < 4; ++i) to[(4 * dd + i) * 64 + lane] = o[dd][i];
    to[D / 4 * 64 + lane] = m;
    to[(D / 4 + 1) * 64 + lane] = l;
  }
  __device__ __forceinline__ void take_over(const float* from) {
    const int lane = threadIdx.x & 63;
    const float om = from[D / 4 * 64 + lane];
    raise(om);
    const float f = m == -kInf ? 1.f : __builtin_amdgcn_exp2f(om - m);
    l = fmaf(from[(D / 4 + 1) * 64 + lane], f, l);
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dd][i] = fmaf(from[(4 * dd + i) * 64 + lane], f, o[dd][i]);
  }
  __device__ __forceinline__ void finish(bool bad) {   // row sums; a slot or page outside the cache makes them NaN
    l = add_lane_xor32(add_lane_xor16(l));
    if (bad) l = __builtin_nanf("");
  }
  __device__ __forceinline__ void store(const SharedArgs& a) const {
    const int grp = (threadIdx.x & 63) >> 4;
    if (place < 0) return;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) *reinterpret_cast<f32x4*>(a.acc + (int64_t)place * D + 16 * dd + 4 * grp) = o[dd];
    if (grp == 0) { a.m[place] = m; a.l[place] = l; }
  }
};

// NB blocks of queries meet 16 SUB tokens, of which the first `live` are the item's.  k: the rows of K in LDS, v: those of V, scales: their scales (e4m3
// only).  What is read from LDS serves all blocks: with one block a wave the LDS is busy longer than the vector unit.
template <typename T, bool FP8, int D, int SUB, int NB>
__device__ __forceinline__ void attend_step(const SharedArgs& a, QueryBlock<T, FP8, D>* blocks, int live, const bf16x8* k,
                                            const bf16x8* v, const Scales scales) {
  typedef Shape<T, FP8, D> S;
  typedef typename S::P P;
  constexpr int N = 4 * SUB;
  const int lane = threadIdx.x & 63, r = lane & 15, grp = lane >> 4;
  float s[NB][N];
#pragma unroll
  for (int j = 0; j < SUB; ++j) {
    const int tok = 16 * j + r;
    f32x4 st[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) st[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk) {
      const auto kf = __builtin_bit_cast(typename S::kvec, k[tok * S::KC + ((4 * kk + grp) ^ (tok & (S::KC - 1)))]);
#pragma unroll
      for (int n = 0; n < NB; ++n) st[n] = HalfMfma<T>::run(kf, blocks[n].q[kk], st[n]);
    }
    if constexpr (FP8) {
      const f32x4 k4 = *reinterpret_cast<const f32x4*>(scales.k + 16 * j + 4 * grp);
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(scales.log_v + 16 * j + 4 * grp);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][4 * j + i] = fmaf(st[n][i], k4[i], l4[i]);
    } else {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][4 * j + i] = st[n][i];
    }
  }
  float mx[NB];
  bool raise = false;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (live < 16 * SUB) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[n][i] = 16 * (i >> 2) + 4 * grp + (i & 3) < live ? s[n][i] : -kInf;
    }
    mx[n] = s[n][0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx[n] = fmaxf(mx[n], s[n][i]);
    if constexpr (!FP8) mx[n] *= a.scale_log2e;   // the scale is positive: scores stay unscaled until the exponential
    raise |= mx[n] > blocks[n].m + 8.0f;
  }
  if (__any(raise)) {
#pragma unroll
    for (int n = 0; n < NB; ++n) blocks[n].raise(max_lane_xor32(max_lane_xor16(mx[n])));
  }
  typename S::pvec pf[NB][SUB / 2], rest[NB][FP8 ? 1 : SUB / 2];
  float ref[NB], sum[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    ref[n] = blocks[n].m == -kInf ? 0.f : blocks[n].m;   // nothing seen yet: every score here is masked, p = 0
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < SUB; ++j) {
    f32x4 r4;
    if constexpr (FP8) r4 = *reinterpret_cast<const f32x4*>(scales.inverse_v + 16 * j + 4 * grp);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int half = j >> 1, at = 4 * (j & 1) + i;
        if constexpr (FP8) {
          const float w = __builtin_amdgcn_exp2f(s[n][4 * j + i] - ref[n]);
          sum[n][i] = fmaf(w, r4[i], sum[n][i]);
          pf[n][half][at] = (P)w;
        } else {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[n][4 * j + i], a.scale_log2e, -ref[n]));
          sum[n][i] += p;
          const P high = (P)p;
          pf[n][half][at] = high;
          rest[n][half][at] = (P)(p - (float)high);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) blocks[n].l += (sum[n][0] + sum[n][1]) + (sum[n][2] + sum[n][3]);
  // tokens 4 grp + i and 16 + 4 grp + i (of each 32) of dim 16 dd + r: the order P holds them in
#pragma unroll
  for (int dd = 0; dd < D / 16; ++dd) {
#pragma unroll
    for (int half = 0; half < SUB / 2; ++half) {
      s16x4 piece[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int tok = 32 * half + 16 * j + 4 * grp + (r >> 2), c = 2 * dd + ((r & 3) >> 1);
        const char* at = reinterpret_cast<const char*>(v + tok * S::KC + (c ^ (tok & (S::KC - 1)))) + 8 * (r & 1);
        piece[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
      }
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      const s16x8 both = {piece[0][0], piece[0][1], piece[0][2], piece[0][3], piece[1][0], piece[1][1], piece[1][2], piece[1][3]};
      const auto vt = __builtin_bit_cast(typename S::pvec, both);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        blocks[n].o[dd] = HalfMfma<P>::run(vt, pf[n][half], blocks[n].o[dd]);
        if constexpr (!FP8) blocks[n].o[dd] = HalfMfma<P>::run(vt, rest[n][half], blocks[n].o[dd]);
      }
    }
  }
}

// Where the tokens of an item are.  Dense: base + t * c1; paged: through the table row.
template <bool PAGED> struct History {
  const SharedArgs& a;
  int64_t base;
  int table_row;
  bool bad;   // a slot or page outside the cache: nothing there is read
  __device__ __forceinline__ History(const SharedArgs& args, int source, int h) : a(args), table_row(source) {
    bad = source < 0 || source >= a.sources;
    base = (PAGED || bad ? 0 : (int64_t)source * a.c0) + (int64_t)h * a.c2;
    if (bad) table_row = -1;
  }
  __device__ __forceinline__ int block_of(int t) const { return a.page_shift >= 0 ? t >> a.page_shift : t / a.page; }
  __device__ __forceinline__ int page_of(int t) const {   // what the table says, checked when it is used
    return table_row < 0 ? 0 : a.table[(int64_t)table_row * a.max_blocks + block_of(t)];
  }
  // in elements; `page` (paged only): page_of(t)
  __device__ __forceinline__ int64_t offset(int t, int page = 0) {
    if constexpr (PAGED) {
      if (page < 0 || page >= a.pools) { bad = true; page = 0; }
      return base + (int64_t)page * a.c0 + (int64_t)(t - block_of(t) * a.page) * a.c1;
    }
    return base + (int64_t)t * a.c1;
  }
};

// 16 bytes of a V row (or of a K row) to LDS as 16-bit values: piece c of row `tok`, swizzled by the row so that the stores
// and both kinds of read spread over the banks.
template <typename T, bool FP8, int D> __device__ __forceinline__ void stage(bf16x8* rows, int tok, int c, const i32x4 w) {
  constexpr int KC = Shape<T, FP8, D>::KC;
  if constexpr (FP8) {
    rows[tok * KC + ((2 * c) ^ (tok & (KC - 1)))] = __builtin_bit_cast(bf16x8, widen8<T>(w[0], w[1]));
    rows[tok * KC + ((2 * c + 1) ^ (tok & (KC - 1)))] = __builtin_bit_cast(bf16x8, widen8<T>(w[2], w[3]));
  } else {
    rows[tok * KC + (c ^ (tok & (KC - 1)))] = __builtin_bit_cast(bf16x8, w);
  }
}

// The way of K and V rows from memory to LDS: THREADS threads bring TOKENS tokens, consecutive threads consecutive 16-byte
// pieces, so that every load instruction asks for whole cache lines.  Of a paged history, each lane looks one row of its
// wave's up in the table, a tile ahead, and hands its place to the lanes that bring it: the table's latency in front of every
// tile's own cost 55 rows of 128 dims and pages of 16 38 us of attention and join instead of 23.
template <typename T, bool FP8, bool PAGED, int D, int THREADS, int TOKENS, bool STREAM> struct Rows {
  typedef Shape<T, FP8, D> S;
  static constexpr int N = TOKENS * S::ROW16 / THREADS;          // pieces per thread, of K and of V
  static constexpr int NS = !FP8 ? 0 : THREADS >= 2 * TOKENS ? 1 : 2;   // scales per thread (K and V, or one of the two)
  static_assert(N >= 1 && (!FP8 || THREADS >= TOKENS), "a thread has a piece, and a token a thread");
  struct Raw { i32x4 k[N], v[N]; float s[NS > 0 ? NS : 1]; };
  const SharedArgs& a;
  History<PAGED>& history;
  const int t1, thread, row_bytes;
  uint32_t whole[N];
  // paged: rows of a wave per load instruction; the row this lane looks up; what it found for the next tile
  static constexpr int PER = 64 / S::ROW16;
  static_assert(PER * N <= 64 && THREADS % S::ROW16 == 0, "a wave has a lane for each of its rows");
  const int own_row;
  int page = 0, scale_page = 0;
  // `first`: where the first fetch will be
  __device__ __forceinline__ Rows(const SharedArgs& args, History<PAGED>& h, int first, int end, int id)
      : a(args), history(h), t1(end), thread(id), row_bytes((int)args.c1 * S::ES),
        own_row((id >> 6) * PER + (id & 63) % PER + THREADS / S::ROW16 * ((id & 63) / PER % N)) {
    if constexpr (PAGED) {
      look_up(first);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) whole[i] = row_of(i) * row_bytes + 16 * piece_of(i);
    }
  }
  // (a wave by itself looks up consecutive rows, so its lanes have the tokens of their scales already)
  static constexpr bool SCALE_IS_OWN = THREADS == 64;
  __device__ __forceinline__ void look_up(int T0) {
    T0 = T0 < t1 ? T0 : t1 - 1;
    page = history.page_of(T0 + min(own_row, t1 - 1 - T0));
    if constexpr (FP8 && !SCALE_IS_OWN) scale_page = history.page_of(T0 + min(thread % TOKENS, t1 - 1 - T0));
  }
  __device__ __forceinline__ int row_of(int i) const { return (thread + THREADS * i) / S::ROW16; }
  __device__ __forceinline__ int piece_of(int i) const { return (thread + THREADS * i) % S::ROW16; }
  // A history that is read once per step and by one workgroup leaves nothing in the caches that anybody wants: the
  // non-temporal hint (streaming reads run at 6.9 TB/s with it and 6.1 without).
  template <typename V> static __device__ __forceinline__ V load(const V* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
  }
  // tokens from T0 on, cut to the item's; past its end, its last token for every thread.  The next fetch is of `next`.
  __device__ __forceinline__ void fetch(int T0, int next, Raw& x) {
    T0 = T0 < t1 ? T0 : t1 - 1;
    const int last = t1 - 1 - T0;
    if constexpr (PAGED) {
      const int64_t own = history.offset(T0 + min(own_row, last), page);
      const int64_t bytes = own * S::ES;
      const int low = (int)(uint32_t)bytes, high = (int)(bytes >> 32);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int from = (thread & 63) / S::ROW16 + PER * i;
        const int64_t at = (((int64_t)__shfl(high, from, 64) << 32) | (uint32_t)__shfl(low, from, 64)) + 16 * piece_of(i);
        x.k[i] = load(reinterpret_cast<const i32x4*>((const uint8_t*)a.kc + at));
        x.v[i] = load(reinterpret_cast<const i32x4*>((const uint8_t*)a.vc + at));
      }
      if constexpr (FP8) load_scales((SCALE_IS_OWN ? own : history.offset(T0 + min(thread % TOKENS, last), scale_page)) / D, x);
      look_up(next);
    } else {
      const int64_t start = history.offset(T0);
      const uint8_t* krows = (const uint8_t*)a.kc + start * S::ES;
      const uint8_t* vrows = (const uint8_t*)a.vc + start * S::ES;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        uint32_t at = whole[i];
        if (last < TOKENS - 1) at = min(row_of(i), last) * row_bytes + 16 * piece_of(i);
        x.k[i] = load(reinterpret_cast<const i32x4*>(krows + at));
        x.v[i] = load(reinterpret_cast<const i32x4*>(vrows + at));
      }
      if constexpr (FP8) load_scales(start / D + (uint32_t)min(thread % TOKENS, last) * (uint32_t)(row_bytes / D), x);
    }
  }
  __device__ __forceinline__ void load_scales(int64_t at, Raw& x) const {
    if constexpr (NS == 2) { x.s[0] = load(a.ks + at); x.s[1] = load(a.vs + at); }
    if constexpr (NS == 1) x.s[0] = load((thread < TOKENS ? a.ks : a.vs) + at);
  }
  // pieces [first, first + COUNT) of the thread, the first of them belonging to token `base` of the LDS tile's 0
  template <int FIRST, int COUNT> __device__ __forceinline__ void stage_k(const Raw& x, bf16x8* rows) const {
#pragma unroll
    for (int i = FIRST; i < FIRST + COUNT; ++i) stage<T, FP8, D>(rows, row_of(i) - FIRST * THREADS / S::ROW16, piece_of(i), x.k[i]);
  }
  template <int FIRST, int COUNT> __device__ __forceinline__ void stage_v(const Raw& x, int T0, bf16x8* rows) const {
#pragma unroll
    for (int i = FIRST; i < FIRST + COUNT; ++i) {
      i32x4 w = x.v[i];
      if (T0 + row_of(i) >= t1) w = i32x4{0, 0, 0, 0};   // 0 * whatever the last row holds
      stage<typename S::P, FP8, D>(rows, row_of(i) - FIRST * THREADS / S::ROW16, piece_of(i), w);
    }
  }
  __device__ __forceinline__ void stage_scales(const Raw& x, const Scales to) const {
    if constexpr (NS == 2) {
      if (thread < TOKENS) { to.k[thread] = x.s[0] * a.scale_log2e; to.set_v(thread, x.s[1]); }
    }
    if constexpr (NS == 1) {
      if (thread < TOKENS) to.k[thread] = x.s[0] * a.scale_log2e;
      else if (thread < 2 * TOKENS) to.set_v(thread - TOKENS, x.s[0]);
    }
  }
};

// An item of one block of queries against tokens [t0, t1) of one KV head.  A wave works by itself on tiles of 4 KiB of K and
// of V (at least 32 tokens): the next one is on its way to registers while the rows of the current one pass through the
// wave's own LDS, 32 tokens at a time.  The four waves of a workgroup share a long item, taking its tiles round robin (the
// four then read 16 KiB in a row), and their results meet at its end; a short item is one wave's.
template <typename T, bool FP8, bool PAGED, int D, bool LONG>
__device__ __forceinline__ void block_item(const SharedArgs& a, const i32x4 r0, const i32x4 r1, int h, bf16x8* lds, float* lds_scale) {
  typedef Shape<T, FP8, D> S;
  constexpr int TOKENS = 4096 / S::RB > 64 ? 64 : 4096 / S::RB < 32 ? 32 : 4096 / S::RB;
  constexpr int PARTS = TOKENS / kStep, STRIDE = LONG ? 4 * TOKENS : TOKENS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, grp = lane >> 4;
  bf16x8* const lds_k = lds + wave * 2 * kStep * S::KC;
  bf16x8* const lds_v = lds_k + kStep * S::KC;
  const Scales scales{lds_scale + wave * 192, lds_scale + wave * 192 + 64, lds_scale + wave * 192 + 128};
  const int t0 = r1[0] + (LONG ? wave * TOKENS : 0), t1 = r1[1];
  History<PAGED> history(a, PAGED && r1[3] == kOwn ? r0[0] : r1[2], h);
  typedef Rows<T, FP8, PAGED, D, 64, TOKENS, true> Tile;
  Tile tile(a, history, t0, t1, lane);
  typename Tile::Raw raw;
  const bool work = t0 < t1 && (PAGED || !history.bad);   // the same for the whole wave
  if (work) tile.fetch(t0, t0 + STRIDE, raw);
  QueryBlock<T, FP8, D> block;
  block.start(a, r0, r1[3], h, r0[2] * kQueryBlock);
  if (work) {
    for (int T0 = t0; T0 < t1; T0 += STRIDE) {
      typename Tile::Raw now = raw;
      auto part = [&](auto index) __attribute__((always_inline)) {
        constexpr int PART = decltype(index)::value, COUNT = Tile::N / PARTS;
        const int from = T0 + kStep * PART;
        wave_sync();
        tile.template stage_k<PART * COUNT, COUNT>(now, lds_k);
        tile.template stage_v<PART * COUNT, COUNT>(now, T0, lds_v);
        if constexpr (FP8 && PART == 0) tile.stage_scales(now, scales);
        wave_sync();
        if constexpr (PART == PARTS - 1) tile.fetch(T0 + STRIDE, T0 + 2 * STRIDE, raw);
        if (PART == 0 || from < t1) attend_step<T, FP8, D, 2, 1>(a, &block, t1 - from, lds_k, lds_v, scales + kStep * PART);
      };
      part(std::integral_constant<int, 0>{});
      if constexpr (PARTS == 2) part(std::integral_constant<int, 1>{});
    }
  }
  block.finish(__any(history.bad));
  if constexpr (LONG) {   // the four results meet
    float* const share = reinterpret_cast<float*>(lds);
    __syncthreads();
    if (wave > 0) block.hand_over(share + (wave - 1) * block.kShare);
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 0; w < 3; ++w) block.take_over(share + w * block.kShare);
      block.store(a);
    }
    __syncthreads();   // the next item's tiles go where the results met
  } else {
    block.store(a);
  }
}

// A shared item: up to 64 queries of a group against tokens [t0, t1) of one KV head, 128 tokens at a time.  All four waves
// stage the tile (the next one is on its way to registers meanwhile); then each takes NB query blocks against its share of the
// tile's tokens: the waves of one set of blocks share them evenly, and their results meet at the end.  An e4m3 history takes
// two blocks a wave (32 x 16 rows, 5500 shared tokens: 8 % less time than one block), since each is read with three scales per
// token; a 16-bit one takes one block and twice the tokens at a time (6 % less time than two: the weights' second part and the
// wider rows in flight need the registers).
template <typename T, bool FP8, bool PAGED, int D>
__device__ __forceinline__ void shared_item(const SharedArgs& a, const i32x4 r0, const i32x4 r1, int h, bf16x8* lds, float* lds_scale) {
  typedef Shape<T, FP8, D> S;
  typedef QueryBlock<T, FP8, D> Block;
  constexpr int NB = FP8 ? 2 : 1, SUB = FP8 || D > 64 ? 2 : 4, STEP = 16 * SUB;
  bf16x8* const lds_k = lds;
  bf16x8* const lds_v = lds + kShareTile * S::KC;
  const Scales scales{lds_scale, lds_scale + kShareTile, lds_scale + 2 * kShareTile};
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = r1[0], t1 = r1[1];
  const int q0 = r0[2] * kQueryTile, queries = min(r0[1] * a.G - q0, kQueryTile);
  const int sets = (queries > 32 ? 4 : 2) / NB, set = wave & (sets - 1);
  const int tokens = kShareTile / 4 * sets, first = wave / sets * tokens;   // the wave's share of a tile
  History<PAGED> history(a, r1[2], h);
  typedef Rows<T, FP8, PAGED, D, 256, kShareTile, false> Tile;
  Tile tile(a, history, t0, t1, threadIdx.x);
  typename Tile::Raw raw;
  const bool readable = PAGED || !history.bad;
  if (readable) tile.fetch(t0, t0 + kShareTile, raw);
  Block blocks[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) blocks[n].start(a, r0, kShared, h, q0 + 16 * (NB * set + n));
  if (readable) {
    for (int T0 = t0; T0 < t1; T0 += kShareTile) {
      __syncthreads();
      tile.template stage_k<0, Tile::N>(raw, lds_k);
      tile.template stage_v<0, Tile::N>(raw, T0, lds_v);
      if constexpr (FP8) tile.stage_scales(raw, scales);
      __syncthreads();
      tile.fetch(T0 + kShareTile, T0 + 2 * kShareTile, raw);
      for (int row = first; row < first + tokens; row += STEP) {
        const int from = T0 + row;
        if (from >= t1) break;
        attend_step<T, FP8, D, SUB, NB>(a, blocks, t1 - from, lds_k + row * S::KC, lds_v + row * S::KC, scales + row);
      }
    }
  }
  const bool bad = __syncthreads_or(history.bad);   // also: the last tile has been read by all waves
#pragma unroll
  for (int n = 0; n < NB; ++n) blocks[n].finish(bad);
  // the first wave of a set keeps; the others hand over to it, one after the other
  float* const share = reinterpret_cast<float*>(lds) + set * NB * Block::kShare;
  for (int giver = sets; giver < 4; giver += sets) {
    if (wave / sets == giver / sets) {
#pragma unroll
      for (int n = 0; n < NB; ++n) blocks[n].hand_over(share + n * Block::kShare);
    }
    __syncthreads();
    if (wave < sets) {
#pragma unroll
      for (int n = 0; n < NB; ++n) blocks[n].take_over(share + n * Block::kShare);
    }
    __syncthreads();   // the next results, and the next item's tiles, go to the same place
  }
  if (wave < sets) {
#pragma unroll
    for (int n = 0; n < NB; ++n) blocks[n].store(a);
  }
}

// Own parts alone (256 rows of 2000 tokens, 8 KV heads of 64 dims), this launch and the join's 5 us: 184 us in bf16 (5.9 TB/s in
// this one), 119 in e4m3 (4.9).  Both have three waves a SIMD with 4 KiB each of K and of V; a tile of e4m3 is 64 tokens, and
// the next one is asked for when the second half of it has been staged, so that nothing is on its way during the first, while a
// 16-bit tile of 32 tokens is replaced as soon as it has been staged.  (`attend` on the same rows: 162 and 94.)  Shared parts
// alone (32 x 16 rows, 5500 tokens, 23 GFLOP, 90 M exponentials), with the join: 87 us in bf16, 65 in e4m3, bound by LDS reads
// and vector instructions per score (an earlier e4m3 build of 70 us took 45 for loads alone, 56 for arithmetic alone and 65 for
// arithmetic and staging).
template <typename T, bool FP8, bool PAGED, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D <= 64 ? 3 : 2))) shared_attention_kernel(SharedArgs a) {
  typedef Shape<T, FP8, D> S;
  __shared__ bf16x8 lds[2 * kShareTile * S::KC];   // K and V: 32 tokens for each wave, or 128 for the workgroup
  __shared__ __attribute__((aligned(16))) float lds_scale[4 * 192];
  static_assert(4 * QueryBlock<T, FP8, D>::kShare * 4 <= (int)sizeof(lds), "the waves' results fit the tile memory");
  if (!list_fits(a, D)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int32_t* const records = a.schedule + kHeader + kRowInts * a.B;
  const int shared_records = a.schedule[kHShared], long_records = a.schedule[kHLong], short_records = a.schedule[kHShort];
  auto record = [&](int at, i32x4& r0, i32x4& r1) {   // the same in every lane
    const i32x4* rec = reinterpret_cast<const i32x4*>(records + (int64_t)kRecordInts * at);
    auto scalar = [](const i32x4 v) {
      return i32x4{__builtin_amdgcn_readfirstlane(v[0]), __builtin_amdgcn_readfirstlane(v[1]), __builtin_amdgcn_readfirstlane(v[2]),
                   __builtin_amdgcn_readfirstlane(v[3])};
    };
    r0 = scalar(rec[0]);
    r1 = scalar(rec[1]);
  };
  i32x4 r0, r1;
  // The first 2 * shared_blocks workgroups take shared and other items in turn, the rest other items: what runs at the same
  // time on a CU is some of each (shared parts are bound by arithmetic, the others by memory).  A turn is one workgroup for
  // every CU: consecutive workgroups go to the XCDs, their shader engines and CUs in turn, so that a shorter period would
  // give all shared items to some of them (32 x 16 rows, 5500 shared tokens: turns of 256 workgroups take 69 % of the time that
  // turns of 8 take in e4m3, 74 % in bf16).  The grid fills the chip about once and strides over the items: a workgroup without
  // work costs its slot a microsecond or two.
  int block = blockIdx.x;
  if (block < 2 * a.shared_blocks && block % (2 * kTurn) < kTurn) {
    for (int idx = block / (2 * kTurn) * kTurn + block % kTurn; idx < shared_records * a.KH; idx += a.shared_blocks) {
      record(idx / a.KH, r0, r1);
      shared_item<T, FP8, PAGED, D>(a, r0, r1, idx % a.KH, lds, lds_scale);
    }
    return;
  }
  block = block < 2 * a.shared_blocks ? block / (2 * kTurn) * kTurn + block % kTurn : block - a.shared_blocks;
  for (int idx = block; idx < long_records * a.KH; idx += a.other_blocks) {
    record(shared_records + idx / a.KH, r0, r1);
    block_item<T, FP8, PAGED, D, true>(a, r0, r1, idx % a.KH, lds, lds_scale);
  }
  for (int idx = block * 4 + wave; idx < short_records * a.KH; idx += 4 * a.other_blocks) {
    record(shared_records + long_records + idx / a.KH, r0, r1);
    block_item<T, FP8, PAGED, D, false>(a, r0, r1, idx % a.KH, lds, lds_scale);
  }
}

// Joins the partial results of one (row, query head) per wave: weights 2^{m_c - max}, one chunk per lane, read back lane by
// lane; lanes own dims.  The results were written by other XCDs and come from beyond the local L2: what counts is the
// number of dependent loads, so a chunk's maximum and sum are read together with the first results, eight chunks at a time
// (512 rows of 32 heads: 7.5 us; 256 rows: 5.4).
template <typename T, int D>
__global__ void __launch_bounds__(256) shared_combine_kernel(SharedArgs a) {
  constexpr int PER = (D + 63) / 64, BATCH = 8;
  const int lane = threadIdx.x & 63, b = blockIdx.x, qh = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (qh >= a.QH) return;
  T* out = (T*)a.out + ((int64_t)b * a.QH + qh) * D;
  const i32x4 row = *reinterpret_cast<const i32x4*>(a.schedule + kHeader + kRowInts * b);
  if (!list_fits(a, D)) {   // a work list of another batch
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i < D) out[lane + 64 * i] = Elem<T>::store(__builtin_nanf(""));
    return;
  }
  const int n = row[3] > 0 ? row[1] + row[2] : 0;
  const int64_t first = (int64_t)row[0] * a.QH + qh;
  float top = -kInf, lt = 0.f, o[PER] = {};
  for (int c0 = 0; c0 < n; c0 += 64) {
    const int here = min(64, n - c0);
    float v[BATCH][PER];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const float* from = a.acc + (first + (int64_t)(c0 + min(i0 + i, here - 1)) * a.QH) * D;
#pragma unroll
        for (int u = 0; u < PER; ++u) v[i][u] = from[min(lane + 64 * u, D - 1)];
      }
    };
    fetch(0);
    const int64_t mine = first + (int64_t)(c0 + min(lane, here - 1)) * a.QH;
    const float mc = lane < here ? a.m[mine] : -kInf, lc = a.l[mine];
    const float now = fmaxf(top, wave_max(mc)), before = now == -kInf ? 1.f : __builtin_amdgcn_exp2f(top - now);
    const float f = lane >= here ? 0.f : now == -kInf ? 1.f : __builtin_amdgcn_exp2f(mc - now);
    lt = lt * before + (lane < here ? lc * f : 0.f);
    top = now;
#pragma unroll
    for (int u = 0; u < PER; ++u) o[u] *= before;
    for (int i0 = 0; i0 < here; i0 += BATCH) {
      if (i0) fetch(i0);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        // chunks past the last: weight 0, of a value that was read before and is not used
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(i0 + i, 63)));
#pragma unroll
        for (int u = 0; u < PER; ++u)
          if (i0 + i < here) o[u] = fmaf(v[i][u], w, o[u]);
      }
    }
  }
  lt = wave_sum(lt);
#pragma unroll
  for (int u = 0; u < PER; ++u)
    if (lane + 64 * u < D) out[lane + 64 * u] = Elem<T>::store(n > 0 ? o[u] / lt : 0.f);
}

int check_batch(const char* name, int64_t B, int QH, int KH, int D, int64_t capacity) {
  LFM2_REQUIRE(B > 0 && QH > 0 && KH > 0 && capacity > 0, "%s: empty shape", name);
  LFM2_REQUIRE(B <= kMaxRows, "%s: more than %d rows", name, kMaxRows);
  LFM2_REQUIRE(QH % KH == 0, "%s: %d query heads not divisible by %d KV heads", name, QH, KH);
  LFM2_REQUIRE(QH <= 1024, "%s: more than 1024 query heads", name);
  LFM2_REQUIRE(D == 32 || D == 64 || D == 128, "%s: head_dim %d not in {32,64,128}", name, D);
  // (the work list's bound on partial results needs rows x positions / kSplitSlots to stay below its largest chunk)
  LFM2_REQUIRE(capacity <= (1 << 28), "%s: more than 2^28 positions", name);
  return LFM2_OK;
}

}  // namespace

extern "C" {

int64_t lfm2_shared_schedule_size(int64_t B, int64_t capacity, int QH, int KH, int D) {
  if (check_batch("shared_schedule_size", B, QH, KH, D, capacity)) return 0;
  return schedule_ints(B, capacity, QH / KH);
}

int64_t lfm2_shared_attention_workspace(int64_t B, int64_t capacity, int QH, int KH, int D) {
  if (check_batch("shared_attention_workspace", B, QH, KH, D, capacity)) return 0;
  return slot_bounds(B, capacity, QH / KH).slots * QH * (D + 2);
}

int lfm2_shared_schedule(int32_t* schedule, const int32_t* positions, const uint8_t* active, const int32_t* slot_ids,
                         const int32_t* starts, const int32_t* prefix_slots, const int32_t* prefix_lengths, int64_t B,
                         int64_t groups, int64_t capacity, int QH, int KH, int D, void* stream) {
  if (int e = check_batch("shared_schedule", B, QH, KH, D, capacity)) return e;
  LFM2_REQUIRE(schedule && positions && ((uintptr_t)schedule & 15) == 0, "shared_schedule: null or unaligned argument");
  LFM2_REQUIRE(groups > 0 && groups <= kMaxRows, "shared_schedule: 1 to %d groups", kMaxRows);
  LFM2_REQUIRE(starts && prefix_slots && prefix_lengths, "shared_schedule: the groups need bounds, slots and lengths");
  const ScheduleArgs a{schedule, positions, slot_ids, starts, prefix_slots, prefix_lengths, active, capacity, (int)B, (int)groups, QH, KH, QH / KH, D};
  if (B <= 1024 && groups <= 1024) hipLaunchKernelGGL(shared_schedule_kernel<1>, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(shared_schedule_kernel<kMaxRows / 1024>, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
  LFM2_LAUNCH_CHECK();
}

int lfm2_shared_attention(void* out, const void* q, const void* k_cache, const void* v_cache, const float* k_scales, const float* v_scales,
                          const int32_t* schedule, const int32_t* block_table, int64_t max_blocks, int page, float* workspace,
                          int64_t B, int QH, int KH, int D, int64_t capacity, int64_t pools, int64_t c0, int64_t c1, int64_t c2,
                          float scale, int kv_fp8, int dtype, void* stream) {
  if (int e = check_batch("shared_attention", B, QH, KH, D, capacity)) return e;
  LFM2_REQUIRE(out && q && k_cache && v_cache && schedule && workspace, "shared_attention: null argument");
  LFM2_REQUIRE(!kv_fp8 || (k_scales && v_scales), "shared_attention: e4m3 history without scales");
  LFM2_REQUIRE(pools > 0, "shared_attention: empty cache");
  // maxima are taken before the scale, and it is applied with log2(e)
  LFM2_REQUIRE(scale > 0.f && scale * LFM2_LOG2E <= __FLT_MAX__, "shared_attention: scale must be positive and finite, with log2(e) too");
  LFM2_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace | (uintptr_t)schedule) & 15) == 0,
               "shared_attention: tensors must be 16-byte aligned");
  LFM2_REQUIRE(!block_table || (page > 0 && max_blocks > 0 && max_blocks * (int64_t)page >= capacity), "shared_attention: bad page geometry");
  const int align = kv_fp8 ? (D > 16 ? D : 16) : 8;
  LFM2_REQUIRE(c0 % align == 0 && c1 % align == 0 && c2 % align == 0, "shared_attention: cache strides must be multiples of %d elements", align);
  LFM2_REQUIRE(c1 >= 0 && c1 < (1 << 23), "shared_attention: tokens of the cache are more than 2^23 elements apart");   // 128 rows in 31 bits
  SharedArgs a;
  a.out = out; a.q = q; a.kc = k_cache; a.vc = v_cache; a.ks = k_scales; a.vs = v_scales;
  a.schedule = schedule; a.table = block_table;
  const int64_t slots = slot_bounds(B, capacity, QH / KH).slots;
  a.acc = workspace;
  a.m = workspace + slots * QH * D;
  a.l = a.m + slots * QH;
  a.c0 = c0; a.c1 = c1; a.c2 = c2; a.max_blocks = max_blocks; a.pools = pools; a.sources = block_table ? B : pools;
  a.page = page > 0 ? page : 1;
  a.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz((unsigned)a.page) : -1;
  a.B = (int)B; a.QH = QH; a.KH = KH; a.G = QH / KH; a.capacity = (int)capacity;
  a.scale_log2e = scale * LFM2_LOG2E;
  hipStream_t s = (hipStream_t)stream;
  // workgroups: as many as there can be items of either kind, up to a number that fills the chip and then strides
  const int64_t most = slot_bounds(B, capacity, a.G).records * KH;
  a.shared_blocks = most < kTurn ? kTurn : kSharedBlocks;
  a.other_blocks = most < kTurn ? kTurn : kOtherBlocks;
  const dim3 grid((unsigned)(a.shared_blocks + a.other_blocks)), join((unsigned)B, (unsigned)((QH + 3) / 4));
#define SHARED_(T, FP8, PAGED, D_) hipLaunchKernelGGL((shared_attention_kernel<T, FP8, PAGED, D_>), grid, dim3(256), 0, s, a)
#define SHARED_D_(T, D_)                                                                                              \
  do {                                                                                                                \
    if (kv_fp8) { if (block_table) SHARED_(T, true, true, D_); else SHARED_(T, true, false, D_); }                    \
    else { if (block_table) SHARED_(T, false, true, D_); else SHARED_(T, false, false, D_); }                         \
    hipLaunchKernelGGL((shared_combine_kernel<T, D_>), join, dim3(256), 0, s, a);                                     \
  } while (0)
  switch (dtype) {
    case LFM2_DTYPE_BF16:
      if (D == 32) SHARED_D_(__bf16, 32); else if (D == 64) SHARED_D_(__bf16, 64); else SHARED_D_(__bf16, 128);
      break;
    case LFM2_DTYPE_F16:
      if (D == 32) SHARED_D_(_Float16, 32); else if (D == 64) SHARED_D_(_Float16, 64); else SHARED_D_(_Float16, 128);
      break;
    default: LFM2_FAIL(LFM2_ERR_UNSUPPORTED, "shared_attention: dtype %d is not bf16/f16", dtype);
  }
#undef SHARED_D_
#undef SHARED_
  LFM2_LAUNCH_CHECK();
}

}  // extern "C"
