// Decode attention for rows in groups that share the first part of their history (the completions of one prompt): the
// shared positions are read once for all rows of a group, each row's own positions once, and the partial softmaxes joined.
//
// Cache addressing is that of attention.hip: element (slot, pos, head, d) at slot*c0 + pos*c1 + head*c2 + d, the e4m3 scale
// of (slot, pos, head) at that offset divided by D; with a block table c0 is the page stride and pos the in-page index.
#include "lfm2_common.h"
#include <type_traits>

namespace {

constexpr float kInf = __builtin_huge_valf();
constexpr int kTile = 32;                 // history tokens per wave and step
constexpr int kGrain = 4 * kTile;         // chunks are whole steps of the workgroup's four waves
constexpr int kMaxRows = 4096;            // rows and groups the work list holds
constexpr int kSplitSlots = 2048;         // partial results beyond one per row, for the shared and for the own part
constexpr int kSharedItems = 1024;        // workgroup items the shared parts are cut into, if their length allows ...
constexpr int kOwnItems = 2048;           // ... and the rows' own parts

// Queries of one item: a tile of the (row, head) pairs of a group that use one KV head.
constexpr int query_tile(int D) { return D <= 64 ? 64 : 32; }

// ---- the work list (int32), built once per decode step and used by every attention layer
//   header: what the list was built for, number of records, number of shared records
//   one record per row: first partial result, shared chunks, own chunks, length (0: sits out)
//   one record per item: first row, rows, query tile, first partial result's offset within a row, first token, end token,
//   slot or table row that holds them, 1 for a shared part
enum { kHRecords, kHRows, kHCapacity, kHQueryHeads, kHKvHeads, kHDim, kHeader = 16 };
constexpr int kRowInts = 4, kRecordInts = 8;

struct SlotBounds { int64_t slots, records; };
// Upper bounds of the partial results and of the items of a batch, from what the host knows.
SlotBounds slot_bounds(int64_t B, int64_t capacity, int G, int D) {
  const int64_t per_row = (capacity + kGrain - 1) / kGrain;
  const int64_t half = B * per_row < B + kSplitSlots ? B * per_row : B + kSplitSlots;
  const int64_t tile = query_tile(D), tiles = (G + tile - 1) / tile;
  return SlotBounds{2 * half, half * (2 * tiles + 1)};
}
int64_t schedule_ints(int64_t B, int64_t capacity, int G, int D) {
  return kHeader + kRowInts * B + kRecordInts * slot_bounds(B, capacity, G, D).records;
}

struct ScheduleArgs {
  int32_t* schedule;
  const int32_t *positions, *slot_ids, *starts, *prefix_slots, *prefix_lengths;
  const uint8_t* active;
  int64_t capacity;
  int B, groups, QH, KH, D;
};

__device__ __forceinline__ int round_up(int v, int step) { return (v + step - 1) / step * step; }

// Sums and exclusive prefix sums over 1024 threads.
__device__ __forceinline__ int scan_1024(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(x, o, 64);
    if (lane >= o) x += up;
  }
  __syncthreads();
  if (lane == 63) scratch[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    before += w < wave ? scratch[w] : 0;
    all += scratch[w];
  }
  *total = all;
  return before + x - v;
}
__device__ __forceinline__ float sum_1024(float v, float* scratch) { return block_sum<16>(v, scratch); }

__global__ void __launch_bounds__(1024) shared_schedule_kernel(ScheduleArgs a) {
  constexpr int PER = kMaxRows / 1024;
  __shared__ int starts[kMaxRows + 1], length[kMaxRows], extent[kMaxRows];
  __shared__ int scratch[16];
  __shared__ float fscratch[16];
  const int tid = threadIdx.x, G = a.QH / a.KH, tile = query_tile(a.D);
  const int capacity = (int)a.capacity;
  for (int g = tid; g <= a.groups; g += 1024) {
    const int s = a.starts[g];
    starts[g] = s < 0 ? 0 : s > a.B ? a.B : s;
    if (g < a.groups) extent[g] = 0;
  }
  __syncthreads();
  // bounds out of order would give a row to several groups: such a list is marked as nobody's (its users return NaN)
  int disorder = 0;
  for (int g = tid; g < a.groups; g += 1024) disorder |= starts[g] > starts[g + 1];
  if (__syncthreads_or(disorder)) {
    if (tid == 0) a.schedule[kHRows] = -1;
    return;
  }
  // a row's group: the last one that starts at or before it
  int group[PER], shared[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    group[i] = -1;
    shared[i] = 0;
    if (b >= a.B) continue;
    int lo = 0, hi = a.groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (starts[mid] <= b) lo = mid; else hi = mid;
    }
    int len = a.positions[b] < capacity ? a.positions[b] + 1 : capacity;
    if (len < 0 || (a.active && !a.active[b]) || (a.slot_ids && a.slot_ids[b] < 0)) len = 0;
    length[b] = len;
    if (starts[lo] <= b && b < starts[lo + 1] && a.prefix_slots[lo] >= 0) {
      const int p = a.prefix_lengths[lo];
      group[i] = lo;
      shared[i] = p < 0 ? 0 : p > capacity ? capacity : p;
      atomicMax(&extent[lo], len < shared[i] ? len : shared[i]);
    }
  }
  __syncthreads();
  // chunk sizes: enough items to fill the chip, no more partial results than the workspace holds
  float row_tokens = 0.f, own_tokens = 0.f, work = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    if (b >= a.B) continue;
    if (group[i] >= 0) row_tokens += (float)extent[group[i]];
    if (length[b] > shared[i]) own_tokens += (float)(length[b] - shared[i]);
  }
  auto group_tiles = [&](int g) {   // query tiles of a group whose rows share anything
    const int rows = starts[g + 1] - starts[g];
    return extent[g] > 0 && rows > 0 ? (rows * G + tile - 1) / tile : 0;
  };
  for (int g = tid; g < a.groups; g += 1024) work += (float)extent[g] * (float)group_tiles(g);
  row_tokens = sum_1024(row_tokens, fscratch);
  own_tokens = sum_1024(own_tokens, fscratch);
  work = sum_1024(work, fscratch);
  const int own_tiles = (G + tile - 1) / tile;
  auto chunk_of = [&](float slots_tokens, float item_tokens, int items) {
    // one more step than the quotient: the sums are rounded
    const float need = fmaxf(slots_tokens / (float)kSplitSlots, item_tokens * (float)a.KH / (float)items);
    return round_up((int)fminf(need * 1.0001f, 1.0e9f) + 1, kGrain);
  };
  const int shared_chunk = chunk_of(row_tokens, work, kSharedItems);
  const int own_chunk = chunk_of(own_tokens, own_tokens * (float)own_tiles, kOwnItems);
  // places: partial results of every row, then the records of the shared parts and of the own parts
  int slots = 0, own_records = 0;
  int np[PER], ns[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    np[i] = ns[i] = 0;
    if (b >= a.B) continue;
    if (group[i] >= 0) np[i] = (extent[group[i]] + shared_chunk - 1) / shared_chunk;
    if (length[b] > shared[i]) ns[i] = (length[b] - shared[i] + own_chunk - 1) / own_chunk;
    slots += np[i] + ns[i];
    own_records += ns[i] * own_tiles;
  }
  int total, shared_total, own_total;
  int slot = scan_1024(slots, scratch, &total);
  int shared_records = 0;
  for (int i = 0; i < PER; ++i) {
    const int g = tid * PER + i;
    if (g < a.groups) shared_records += (extent[g] + shared_chunk - 1) / shared_chunk * group_tiles(g);
  }
  int record = scan_1024(shared_records, scratch, &shared_total);
  int own_record = shared_total + scan_1024(own_records, scratch, &own_total);
  int32_t* const records = a.schedule + kHeader + kRowInts * a.B;
  auto put = [&](int at, int row, int rows, int qt, int offset, int t0, int t1, int source, int is_shared) {
    i32x4* r = reinterpret_cast<i32x4*>(records + (int64_t)kRecordInts * at);
    r[0] = i32x4{row, rows, qt, offset};
    r[1] = i32x4{t0, t1, source, is_shared};
  };
  for (int i = 0; i < PER; ++i) {
    const int g = tid * PER + i;
    if (g >= a.groups) break;
    const int tiles = group_tiles(g);
    for (int t0 = 0, c = 0; tiles > 0 && t0 < extent[g]; t0 += shared_chunk, ++c)
      for (int qt = 0; qt < tiles; ++qt)
        put(record++, starts[g], starts[g + 1] - starts[g], qt, c, t0, min(t0 + shared_chunk, extent[g]), a.prefix_slots[g], 1);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = tid * PER + i;
    if (b >= a.B) continue;
    int32_t* r = a.schedule + kHeader + kRowInts * b;
    r[0] = slot; r[1] = np[i]; r[2] = ns[i]; r[3] = length[b];
    slot += np[i] + ns[i];
    const int source = a.slot_ids ? a.slot_ids[b] : b;
    for (int c = 0; c < ns[i]; ++c)
      for (int qt = 0; qt < own_tiles; ++qt) {
        const int t0 = shared[i] + c * own_chunk;
        put(own_record++, b, 1, qt, np[i] + c, t0, min(t0 + own_chunk, length[b]), source, 0);
      }
  }
  if (tid == 0) {
    a.schedule[kHRecords] = shared_total + own_total;
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

struct SharedArgs {
  void* out;
  const void *q, *kc, *vc;
  const float *ks, *vs;
  const int32_t *schedule, *table;
  float *acc, *m, *l;          // partial results: [slot][query head][D], [slot][query head] twice
  int64_t c0, c1, c2, max_blocks, pools, sources;   // pools: slots or pages; sources: slots or table rows
  int page, page_shift, B, QH, KH, G, capacity;
  float scale_log2e;
};
__device__ __forceinline__ bool list_fits(const SharedArgs& a, int D) {
  const int32_t* s = a.schedule;
  return s[kHRows] == a.B && s[kHCapacity] == a.capacity && s[kHQueryHeads] == a.QH && s[kHKvHeads] == a.KH && s[kHDim] == D;
}

// One item: MT * 16 queries against tokens [t0, t1) of one KV head.  The four waves take the tokens in tiles of 32, round
// robin; lane % 16 is the lane's query throughout (grp = lane / 16):
//   S^T  = K . Q^T   (A = 16 tokens x 32 dims, B = 32 dims x 16 queries): the lane gets tokens 4 grp + i of its query;
//   O^T += V^T . P^T (A = V^T through the transposing read of the row-major tile, B = P straight from the S^T registers).
// A lane loads 16 consecutive bytes of a K row; which dims those are only has to match between K and Q, so an e4m3 lane
// takes dims 64 i + 16 grp .. + 15 and uses them as two operands.  K goes from memory to the operand registers; V passes
// through the wave's own LDS tile (no barrier: nothing is shared between waves until the end).
// The running maximum is raised only when a score exceeds it by more than 8 (powers of two), so most tiles need no
// rescaling: p <= 2^8 fits every type used here and the reference point cancels in the end.
template <typename T, bool FP8, int D> struct Shape {
  typedef std::conditional_t<FP8, __bf16, T> P;   // type of P and V: P carries the V scale, which fp16 could not hold
  static constexpr int ES = FP8 ? 1 : 2, RB = D * ES;
  static constexpr int KK = D / 32;                                   // products per 16 x 16 scores
  static constexpr int KP = FP8 && D == 32 ? 1 : RB / 64;             // 16-byte pieces of a K row per lane
  static constexpr int VP = RB / 32;                                  // 16-byte pieces of the V tile per lane
  static constexpr int KC = D / 8;                                    // 16-byte pieces of a V row in LDS
  static constexpr int QT = query_tile(D) / 16;
};

template <typename T, bool FP8, bool PAGED, int D, int MT>
__device__ __forceinline__ void attend_item(const SharedArgs& a, const i32x4 r0, const i32x4 r1, int h, bf16x8* lds_v,
                                            float (*lds_scale)[kTile], float* lds_o, float (*lds_m)[64], float (*lds_l)[64]) {
  typedef Shape<T, FP8, D> S;
  typedef typename HalfMfma<T>::vec8 kvec;
  typedef typename HalfMfma<typename S::P>::vec8 pvec;
  typedef typename S::P P;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, grp = lane >> 4;
  const int row0 = r0[0], rows = r0[1], q0 = r0[2] * query_tile(D), offset = r0[3];
  const int t0 = r1[0], t1 = r1[1], source = PAGED && !r1[3] ? row0 : r1[2], total = rows * a.G;
  const int32_t* const row_records = a.schedule + kHeader;
  bool bad = source < 0 || source >= a.sources;
  const int64_t base = (PAGED || bad ? 0 : (int64_t)source * a.c0) + (int64_t)h * a.c2;

  // ---- the queries
  kvec qf[MT][S::KK];
  int limit[MT], least = t1;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    int qi = q0 + 16 * mt + r;
    qi = qi < total ? qi : total - 1;
    const int b = row0 + qi / a.G;
    const T* src = (const T*)a.q + ((int64_t)b * a.QH + h * a.G + qi % a.G) * D;
#pragma unroll
    for (int kk = 0; kk < S::KK; ++kk) {
      const int dim = !FP8 || D == 32 ? 32 * kk + 8 * grp : 64 * (kk >> 1) + 16 * grp + 8 * (kk & 1);
      qf[mt][kk] = *reinterpret_cast<const kvec*>(src + dim);
    }
    const int len = row_records[kRowInts * b + 3];
    limit[mt] = len > 0 && len < t1 ? len : t1;   // a row that sits out computes something that is never stored
    least = limit[mt] < least ? limit[mt] : least;
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));

  f32x4 o[MT][D / 16];
  float m[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -kInf;
    l[mt] = 0.f;
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd) o[mt][dd] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto token_offset = [&](int t) -> int64_t {   // elements, for a token of the item
    if (PAGED) {
      const int blk = a.page_shift >= 0 ? t >> a.page_shift : t / a.page;
      int pool = bad ? 0 : a.table[(int64_t)source * a.max_blocks + blk];
      if (pool < 0 || pool >= a.pools) { bad = true; pool = 0; }
      return base + (int64_t)pool * a.c0 + (int64_t)(t - blk * a.page) * a.c1;
    }
    return base + (int64_t)t * a.c1;
  };
  struct Raw { i32x4 k[2][S::KP], v[S::VP]; float ks, vs; };
  auto fetch = [&](int T0, Raw& x) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      int t = T0 + 16 * j + r;
      t = t < t1 ? t : t1 - 1;
      const uint8_t* row = (const uint8_t*)a.kc + token_offset(t) * S::ES;
      if constexpr (FP8 && D == 32) {
        const i32x2 half = *reinterpret_cast<const i32x2*>(row + 8 * grp);
        x.k[j][0] = i32x4{half[0], half[1], 0, 0};
      } else {
#pragma unroll
        for (int i = 0; i < S::KP; ++i) x.k[j][i] = *reinterpret_cast<const i32x4*>(row + 64 * i + 16 * grp);
      }
    }
#pragma unroll
    for (int u = 0; u < S::VP; ++u) {
      constexpr int per_row = S::RB / 16;
      const int piece = lane + 64 * u;
      int t = T0 + piece / per_row;
      t = t < t1 ? t : t1 - 1;
      x.v[u] = *reinterpret_cast<const i32x4*>((const uint8_t*)a.vc + token_offset(t) * S::ES + 16 * (piece % per_row));
    }
    if constexpr (FP8) {
      int t = T0 + (lane & 31);
      t = t < t1 ? t : t1 - 1;
      const int64_t at = token_offset(t) / D;
      x.ks = a.ks[at];
      x.vs = a.vs[at];
    }
  };

  const int first = t0 + wave * kTile;
  Raw raw;
  if (first < t1 && !(bad && !PAGED)) {
    fetch(first, raw);
    for (int T0 = first; T0 < t1; T0 += kGrain) {
      const bool edge = T0 + kTile > least;
      // ---- this tile: V to LDS, K to operands
      kvec kf[2][S::KK];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int kk = 0; kk < S::KK; ++kk) {
          if constexpr (!FP8) kf[j][kk] = __builtin_bit_cast(kvec, raw.k[j][kk]);
          else if constexpr (D == 32) kf[j][kk] = widen8<T>(raw.k[j][0][0], raw.k[j][0][1]);
          else kf[j][kk] = widen8<T>(raw.k[j][kk >> 1][2 * (kk & 1)], raw.k[j][kk >> 1][2 * (kk & 1) + 1]);
        }
#pragma unroll
      for (int u = 0; u < S::VP; ++u) {
        constexpr int per_row = S::RB / 16;
        const int piece = lane + 64 * u, tok = piece / per_row, c = piece % per_row;
        i32x4 w = raw.v[u];
        if (T0 + tok >= t1) w = i32x4{0, 0, 0, 0};   // 0 * whatever the last row holds
        if constexpr (FP8) {
          const bf16x8 lo = widen8<__bf16>(w[0], w[1]), hi = widen8<__bf16>(w[2], w[3]);
          lds_v[tok * S::KC + ((2 * c) ^ (tok & (S::KC - 1)))] = lo;
          lds_v[tok * S::KC + ((2 * c + 1) ^ (tok & (S::KC - 1)))] = hi;
        } else {
          lds_v[tok * S::KC + (c ^ (tok & (S::KC - 1)))] = __builtin_bit_cast(bf16x8, w);
        }
      }
      float ksc[8], vsc[8];
      if constexpr (FP8) {
        if (lane < kTile) { lds_scale[0][lane] = raw.ks * a.scale_log2e; lds_scale[1][lane] = raw.vs; }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const f32x4 k4 = *reinterpret_cast<const f32x4*>(&lds_scale[0][16 * j + 4 * grp]);
          const f32x4 v4 = *reinterpret_cast<const f32x4*>(&lds_scale[1][16 * j + 4 * grp]);
#pragma unroll
          for (int i = 0; i < 4; ++i) { ksc[4 * j + i] = k4[i]; vsc[4 * j + i] = v4[i]; }
        }
      }
      if (T0 + kGrain < t1) fetch(T0 + kGrain, raw);

      // ---- scores and probabilities of every query block
      pvec pf[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float s[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          f32x4 st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < S::KK; ++kk) st = HalfMfma<T>::run(kf[j][kk], qf[mt][kk], st);
#pragma unroll
          for (int i = 0; i < 4; ++i) s[4 * j + i] = st[i] * (FP8 ? ksc[4 * j + i] : a.scale_log2e);
        }
        if (edge) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * j + i] = T0 + 16 * j + 4 * grp + i < limit[mt] ? s[4 * j + i] : -kInf;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        if (__any(mx > m[mt] + 8.0f)) {
          mx = max_lane_xor32(max_lane_xor16(mx));
          const float mnew = fmaxf(m[mt], mx);
          const float alpha = mnew == -kInf ? 1.f : __builtin_amdgcn_exp2f(m[mt] - mnew);
          m[mt] = mnew;
          l[mt] *= alpha;
#pragma unroll
          for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[mt][dd][i] *= alpha;
        }
        const float ref = m[mt] == -kInf ? 0.f : m[mt];   // nothing seen yet: every score here is masked, p = 0
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = __builtin_amdgcn_exp2f(s[i] - ref);
          sum += p;
          pf[mt][i] = (P)(FP8 ? p * vsc[i] : p);
        }
        l[mt] += sum;
      }
      // ---- O^T += V^T . P^T: tokens 4 grp + i and 16 + 4 grp + i of dim 16 dd + r, the order P holds them in
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) {
        s16x4 half[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int tok = 16 * j + 4 * grp + (r >> 2), c = 2 * dd + ((r & 3) >> 1);
          const char* piece = reinterpret_cast<const char*>(&lds_v[tok * S::KC + (c ^ (tok & (S::KC - 1)))]) + 8 * (r & 1);
          half[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)piece);
        }
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const s16x8 both = {half[0][0], half[0][1], half[0][2], half[0][3], half[1][0], half[1][1], half[1][2], half[1][3]};
        const pvec vf = __builtin_bit_cast(pvec, both);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][dd] = HalfMfma<P>::run(vf, pf[mt], o[mt][dd]);
      }
    }
  }

  // ---- the four waves' partial results meet: statistics first, then one query block of O at a time
  bad = __any(bad);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] = add_lane_xor32(add_lane_xor16(l[mt]));
    if (bad) l[mt] = __builtin_nanf("");   // a slot or page outside the cache
    if (grp == 0) { lds_m[wave][16 * mt + r] = m[mt]; lds_l[wave][16 * mt + r] = l[mt]; }
  }
  __syncthreads();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int q = 16 * mt + r;
    const float mm = fmaxf(fmaxf(lds_m[0][q], lds_m[1][q]), fmaxf(lds_m[2][q], lds_m[3][q]));
    const float f = mm == -kInf ? 0.f : __builtin_amdgcn_exp2f(m[mt] - mm);
#pragma unroll
    for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_o[(wave * 16 + r) * (D + 4) + 16 * dd + 4 * grp + i] = o[mt][dd][i] * f;
    __syncthreads();
    for (int at = threadIdx.x; at < 16 * (D / 4); at += 256) {
      const int query = at / (D / 4), d = 4 * (at % (D / 4)), qi = q0 + 16 * mt + query;
      if (qi < total) {
        const int b = row0 + qi / a.G;
        const int32_t* row = row_records + kRowInts * b;
        if (row[3] > 0) {
          f32x4 sum = *reinterpret_cast<const f32x4*>(&lds_o[query * (D + 4) + d]);
#pragma unroll
          for (int w = 1; w < 4; ++w) sum += *reinterpret_cast<const f32x4*>(&lds_o[(w * 16 + query) * (D + 4) + d]);
          const int64_t at_row = (int64_t)(row[0] + offset) * a.QH + h * a.G + qi % a.G;
          *reinterpret_cast<f32x4*>(a.acc + at_row * D + d) = sum;
          if (d == 0) {
            const int qq = 16 * mt + query;
            const float top = fmaxf(fmaxf(lds_m[0][qq], lds_m[1][qq]), fmaxf(lds_m[2][qq], lds_m[3][qq]));
            float lt = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) lt += lds_l[w][qq] * (top == -kInf ? 1.f : __builtin_amdgcn_exp2f(lds_m[w][qq] - top));
            a.m[at_row] = top;
            a.l[at_row] = lt;
          }
        }
      }
    }
    __syncthreads();
  }
}

template <typename T, bool FP8, bool PAGED, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) shared_attention_kernel(SharedArgs a) {
  typedef Shape<T, FP8, D> S;
  __shared__ bf16x8 lds_v[4][kTile * S::KC];
  __shared__ __attribute__((aligned(16))) float lds_scale[4][2][kTile];
  __shared__ __attribute__((aligned(16))) float lds_o[4 * 16 * (D + 4)];
  __shared__ float lds_m[4][64], lds_l[4][64];
  if (!list_fits(a, D)) return;
  const int wave = threadIdx.x >> 6;
  const int32_t* const records = a.schedule + kHeader + kRowInts * a.B;
  const int items = a.schedule[kHRecords] * a.KH;
  for (int idx = blockIdx.x; idx < items; idx += gridDim.x) {
    const i32x4* rec = reinterpret_cast<const i32x4*>(records + (int64_t)kRecordInts * (idx / a.KH));
    const i32x4 r0 = rec[0], r1 = rec[1];
    const int h = idx % a.KH;
    const int queries = min(r0[1] * a.G - r0[2] * query_tile(D), query_tile(D));
    if (queries <= 16) attend_item<T, FP8, PAGED, D, 1>(a, r0, r1, h, lds_v[wave], lds_scale[wave], lds_o, lds_m, lds_l);
    else if (queries <= 32 || S::QT == 2) attend_item<T, FP8, PAGED, D, 2>(a, r0, r1, h, lds_v[wave], lds_scale[wave], lds_o, lds_m, lds_l);
    else attend_item<T, FP8, PAGED, D, S::QT>(a, r0, r1, h, lds_v[wave], lds_scale[wave], lds_o, lds_m, lds_l);
  }
}

// Joins the partial results of one (row, query head) per wave: weights 2^{m_c - max}, one chunk per lane, read back lane by
// lane; lanes own dims.
template <typename T, int D>
__global__ void __launch_bounds__(256) shared_combine_kernel(SharedArgs a) {
  constexpr int PER = (D + 63) / 64;
  const int lane = threadIdx.x & 63, b = blockIdx.x, qh = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (qh >= a.QH) return;
  T* out = (T*)a.out + ((int64_t)b * a.QH + qh) * D;
  if (!list_fits(a, D)) {   // a work list of another batch
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 64 * i < D) out[lane + 64 * i] = Elem<T>::store(__builtin_nanf(""));
    return;
  }
  const i32x4 row = *reinterpret_cast<const i32x4*>(a.schedule + kHeader + kRowInts * b);
  const int n = row[3] > 0 ? row[1] + row[2] : 0;
  const int64_t first = (int64_t)row[0] * a.QH + qh;
  float top = -kInf;
  for (int c = lane; c < n; c += 64) top = fmaxf(top, a.m[first + (int64_t)c * a.QH]);
  top = wave_max(top);
  float lt = 0.f, o[PER] = {};
  for (int c0 = 0; c0 < n; c0 += 64) {
    const int c = c0 + lane;
    float f = 0.f;
    if (c < n) {
      const float mc = a.m[first + (int64_t)c * a.QH], lc = a.l[first + (int64_t)c * a.QH];
      f = top == -kInf ? 1.f : __builtin_amdgcn_exp2f(mc - top);
      lt = fmaf(lc, f, lt);
    }
    const int here = min(64, n - c0);
    for (int i = 0; i < here; ++i) {
      const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i));
#pragma unroll
      for (int u = 0; u < PER; ++u)
        if (lane + 64 * u < D) o[u] = fmaf(a.acc[(first + (int64_t)(c0 + i) * a.QH) * D + lane + 64 * u], w, o[u]);
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
  return schedule_ints(B, capacity, QH / KH, D);
}

int64_t lfm2_shared_attention_workspace(int64_t B, int64_t capacity, int QH, int KH, int D) {
  if (check_batch("shared_attention_workspace", B, QH, KH, D, capacity)) return 0;
  return slot_bounds(B, capacity, QH / KH, D).slots * QH * (D + 2);
}

int lfm2_shared_schedule(int32_t* schedule, const int32_t* positions, const uint8_t* active, const int32_t* slot_ids,
                         const int32_t* starts, const int32_t* prefix_slots, const int32_t* prefix_lengths, int64_t B,
                         int64_t groups, int64_t capacity, int QH, int KH, int D, void* stream) {
  if (int e = check_batch("shared_schedule", B, QH, KH, D, capacity)) return e;
  LFM2_REQUIRE(schedule && positions && ((uintptr_t)schedule & 15) == 0, "shared_schedule: null or unaligned argument");
  LFM2_REQUIRE(groups > 0 && groups <= kMaxRows, "shared_schedule: 1 to %d groups", kMaxRows);
  LFM2_REQUIRE(starts && prefix_slots && prefix_lengths, "shared_schedule: the groups need bounds, slots and lengths");
  const ScheduleArgs a{schedule, positions, slot_ids, starts, prefix_slots, prefix_lengths, active, capacity, (int)B, (int)groups, QH, KH, D};
  hipLaunchKernelGGL(shared_schedule_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, a);
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
  LFM2_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out | (uintptr_t)workspace | (uintptr_t)schedule) & 15) == 0,
               "shared_attention: tensors must be 16-byte aligned");
  LFM2_REQUIRE(!block_table || (page > 0 && max_blocks > 0 && max_blocks * (int64_t)page >= capacity), "shared_attention: bad page geometry");
  const int align = kv_fp8 ? (D > 16 ? D : 16) : 8;
  LFM2_REQUIRE(c0 % align == 0 && c1 % align == 0 && c2 % align == 0, "shared_attention: cache strides must be multiples of %d elements", align);
  SharedArgs a;
  a.out = out; a.q = q; a.kc = k_cache; a.vc = v_cache; a.ks = k_scales; a.vs = v_scales;
  a.schedule = schedule; a.table = block_table;
  const int64_t slots = slot_bounds(B, capacity, QH / KH, D).slots;
  a.acc = workspace;
  a.m = workspace + slots * QH * D;
  a.l = a.m + slots * QH;
  a.c0 = c0; a.c1 = c1; a.c2 = c2; a.max_blocks = max_blocks; a.pools = pools; a.sources = block_table ? B : pools;
  a.page = page > 0 ? page : 1;
  a.page_shift = (a.page & (a.page - 1)) == 0 ? __builtin_ctz((unsigned)a.page) : -1;
  a.B = (int)B; a.QH = QH; a.KH = KH; a.G = QH / KH; a.capacity = (int)capacity;
  a.scale_log2e = scale * LFM2_LOG2E;
  hipStream_t s = (hipStream_t)stream;
  const int64_t bound = slot_bounds(B, capacity, a.G, D).records * KH;
  const dim3 grid((unsigned)(bound < 1024 ? bound : 1024)), join((unsigned)B, (unsigned)((QH + 3) / 4));
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
