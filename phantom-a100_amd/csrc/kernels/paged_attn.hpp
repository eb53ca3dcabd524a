// Attention of each sequence's new tokens over its pages.
//
// New token i of a sequence of `length` tokens, count of them new, sees the keys at positions up to
// length - count + i (causal) or all of them: O = sum_j softmax_j(q . k_j / sqrt(D)) v_j. Query head h reads
// key/value head h / group. A token that sees no key gets zeros; one whose visible scores are all -inf has a softmax of
// NaN, as the formula has it.
#pragma once

#include "fa_mfma.hpp"
#include "paged_cache.hpp"

namespace pa {

struct RowsQ {
  const void* q;
  void* o;
  int64_t q_token, q_head, o_token, o_head;   // strides in elements
  int group, heads;                            // query heads per key/value head, and query heads
};

// What a workgroup leaves for the join: a part of a tile that an earlier workgroup began (slot 0; kPartEnds if
// it is the tile's last part), a tile begun and not ended (slot 1).
struct PartRecord {
  int seq, head, tile, flags;
};
constexpr int kPartContinues = 1, kPartEnds = 2, kPartBegins = 4;

struct AttnWork {
  TileShape tiles;
  int min_units;       // a workgroup takes at least so many units of work
  int whole, causal;
  float scale_log2;
  PartRecord* records;
  float* parts;        // [workgroup][slot][row][D], then the rows' maxima and sums [workgroup][slot][2][row]
};

// Workspace of a call: a record and two slots of `rows` rows for each workgroup.
__host__ __device__ __forceinline__ int64_t attn_record_bytes(int64_t wgs) { return (wgs * sizeof(PartRecord) + 255) / 256 * 256; }
__host__ __device__ __forceinline__ int64_t attn_workspace(int64_t wgs, int rows, int d) {
  return attn_record_bytes(wgs) + wgs * 2 * rows * (d + 2) * (int64_t)sizeof(float);
}
__device__ __forceinline__ float* part_rows(const AttnWork& w, int wg, int slot, int rows, int d) {
  return w.parts + ((int64_t)wg * 2 + slot) * rows * d;
}
__device__ __forceinline__ float* part_stats(const AttnWork& w, int wgs, int wg, int slot, int rows, int d) {
  return w.parts + (int64_t)wgs * 2 * rows * d + ((int64_t)wg * 2 + slot) * 2 * rows;
}

// Row r of a tile, whichever tile it is: its token and its head among the tile's.
struct InTile {
  int token, head;
};
__device__ __forceinline__ InTile in_tile(const TileShape& t, int r) { return {r / t.heads, r % t.heads}; }
// The key/value head and the part of its group that a tile's `head` stands for.
__device__ __forceinline__ void split_head(const TileShape& t, int head, int& kv_head, int& part) {
  kv_head = t.splits == 1 ? head : head / t.splits;
  part = t.splits == 1 ? 0 : head % t.splits;
}
// The row's new token among the sequence's and its query head; false if the tile has no such row.
__device__ __forceinline__ bool tile_row(const TileShape& t, const SeqRows& s, int head, int tile, InTile r, int& token, int& hq) {
  int kv_head, part;
  split_head(t, head, kv_head, part);
  const int g = part * t.heads + r.head;
  token = tile * t.tokens + r.token;
  hq = kv_head * t.group + g;
  return r.token < t.tokens && token < s.count && g < t.group;
}

// Wave-uniform values in scalar registers: the walk and its branches are the same in every lane, which the
// compiler cannot see where they come from LDS.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(uint32_t)uniform((int)(uint32_t)x) | (int64_t)uniform((int)(x >> 32)) << 32;
}
__device__ __forceinline__ float uniform_f(float x) { return __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, x))); }
__device__ __forceinline__ SeqRows uniform(SeqRows s) { return {uniform(s.first), uniform(s.count), uniform(s.length)}; }

// The workgroup's number `wg` among the shares and, where it has a share, its walk (false: it has none). All
// threads of the workgroup take part; `lds` holds 10 numbers. by_xcd: shares that follow each other go to one
// XCD, whose L2 then serves the tiles of a head together.
template <int THREADS>
__device__ __forceinline__ bool start_walk(const PagedCache& c, const AttnWork& w, bool by_xcd, int64_t* lds, int& wg, WorkWalk& walk) {
  const int heads = c.heads * w.tiles.splits, tid = (int)threadIdx.x, lane = tid % kWave;
  const int per = (c.seqs + THREADS - 1) / THREADS, s0 = min(tid * per, c.seqs), s1 = min(s0 + per, c.seqs);
  auto units = [&](int s) -> int64_t {
    const SeqRows r = load_seq(c, s);
    return heads * tiles_cost(r, w.tiles, w.causal, tiles_of(r, w.tiles));
  };
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += units(s);
  int64_t upto = mine;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t other = __shfl_up(upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == kWave - 1) lds[tid / kWave] = upto;
  __syncthreads();
  int64_t total = 0, before = upto - mine;
#pragma unroll
  for (int i = 0; i < THREADS / kWave; ++i) {
    if (i < tid / kWave) before += lds[i];
    total += lds[i];
  }
  total = uniform(total);
  const int64_t most = total / w.min_units;
  const int active = most < 1 ? 1 : most < (int64_t)gridDim.x ? (int)most : (int)gridDim.x;
  wg = by_xcd && active == (int)gridDim.x ? xcd_remap((int)blockIdx.x, active) : (int)blockIdx.x;
  if (wg >= active || total == 0) return false;
  const int64_t at = share_of(total, active, wg), end = share_of(total, active, wg + 1);
  // The thread whose sequences hold `at` looks for the one that does.
  if (before <= at && at < before + mine) {
    int s = s0;
    for (int64_t u; s + 1 < s1 && before + (u = units(s)) <= at; ++s) before += u;
    lds[8] = before;
    lds[9] = s;
  }
  __syncthreads();
  walk = WorkWalk{w.tiles, c.seqs, heads, c.capacity, w.causal != 0, w.whole != 0, at, end, uniform(lds[8]), uniform((int)lds[9])};
  return true;
}

// ---- Eight or sixteen codes as 16-bit matrix operands (exact) ----
// Pairs of f16 or bf16 in a dword.
template <typename P> __device__ __forceinline__ unsigned pack16(P x) { return __builtin_bit_cast(unsigned, x); }
// Four codes of one dword.
__device__ __forceinline__ void widen4(unsigned w, e4m3*, f16*, unsigned& lo, unsigned& hi) {
  lo = pack16(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, false));
  hi = pack16(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, true));
}
__device__ __forceinline__ void widen4(unsigned w, e4m3*, bf16*, unsigned& lo, unsigned& hi) {
  lo = pack16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, false));
  hi = pack16(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.f, true));
}
// int8 in fp16: 1024 + (x + 128) is 0x6400 with the biased byte as its low bits; 1152 less is x.
__device__ __forceinline__ void widen4(unsigned w, i8*, f16*, unsigned& lo, unsigned& hi) {
  const unsigned u = w ^ 0x80808080u;
  const f16x2 bias = {(f16)1152.f, (f16)1152.f};
  lo = pack16(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u)) - bias);
  hi = pack16(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u)) - bias);
}
__device__ __forceinline__ void widen4(unsigned w, i8*, bf16*, unsigned& lo, unsigned& hi) {
  const bf16x2 a = {(bf16)(float)(int8_t)w, (bf16)(float)(int8_t)(w >> 8)};
  const bf16x2 b = {(bf16)(float)(int8_t)(w >> 16), (bf16)(float)(int8_t)(w >> 24)};
  lo = pack16(a), hi = pack16(b);
}
// The 16 codes of a lane as two operands of 8.
template <typename C, typename T>
__device__ __forceinline__ void widen16(u32x4 w, u32x4& a, u32x4& b) {
  unsigned x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) widen4(w[i], static_cast<C*>(nullptr), static_cast<T*>(nullptr), x[2 * i], x[2 * i + 1]);
  a = u32x4{x[0], x[1], x[2], x[3]};
  b = u32x4{x[4], x[5], x[6], x[7]};
}

// Largest magnitude, as its bits, of pairs of 16-bit values so far; not finite iff it has all exponent bits.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u16x2 max_bits(u16x2 acc, u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_elementwise_max(acc, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  return acc;
}
template <typename T> constexpr unsigned short kInfBits = 0;
template <> constexpr unsigned short kInfBits<f16> = 0x7c00;
template <> constexpr unsigned short kInfBits<bf16> = 0x7f80;

// c plus a pair of 16-bit values.
__device__ __forceinline__ float add_pair(unsigned x, float c, f16*) {
  return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, x), f16x2{(f16)1.f, (f16)1.f}, c, false);
}
__device__ __forceinline__ float add_pair(unsigned x, float c, bf16*) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), bf16x2{(bf16)1.f, (bf16)1.f}, c, false);
}

// Maxima that pass a NaN on: fmaxf first quiets each operand, an instruction apiece. (A row with a NaN score is NaN,
// whatever its reference.)
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Least maximum of a row that sees a key: -inf is for rows that see none. (P is 0 at a score of -inf against it too, and
// the largest finite score's is at least 1: a sum of 0 is of no key or of scores that are all -inf.)
constexpr float kLowest = -3.402823466e38f;
// A row's result x / sum, for a row of maximum m.
__device__ __forceinline__ float row_result(float x, float m, float sum) {
  return sum == 0.f ? (m == -INFINITY ? 0.f : NAN) : x / sum;
}

// x over the lanes of equal lane % 16.
__device__ __forceinline__ float groups_max(float x) { x = fmaxf(x, partner16(x)); return fmaxf(x, partner32(x)); }
__device__ __forceinline__ float groups_sum(float x) { x += partner16(x); return x + partner32(x); }

// fp16 over an 8-bit cache: P times a value's scale goes into a 16-bit product, whatever the scales are, so each row's O
// is held in a unit of its own, and its P times scale is divided by that. The unit follows what the row itself gives
// weight: it starts at kUnitLeast, becomes 2^-8 of the row's largest weight P |scale| when that outgrows it by 2^15 (an
// fp16 reaches 65504), and falls with the row's other sums when its maximum rises. So it never exceeds 2^-8 of the
// largest weight, what a key loses below fp16's normal range is at most 2^-33 of that, and neither a key that the row
// does not see nor a large value that it gives no weight costs it bits.
constexpr float kUnitLeast = 0x1p-100f, kUnitMost = 0x1p120f, kUnitRoom = 0x1p15f;
// The unit of a row, `unit` so far and at least kUnitLeast, whose largest weight is `top`. An infinite weight takes the
// largest unit: the infinity stays one in each dim, and no finite weight becomes another beside it. (A NaN leaves the unit,
// and makes the row NaN in any.)
__device__ __forceinline__ float unit_for(float unit, float top) {
  return top > unit * kUnitRoom ? fminf(top * 0x1p-8f, kUnitMost) : fmaxf(unit, kUnitLeast);
}

// ---- Few rows a tile: single tokens, and the few tokens of one ----
//
// A tile has 16 NB rows; its keys go past once, and what bounds the kernel is reading them: 4 D bytes (2 D in 8
// bits) for 4 D x rows operations. The waves of a workgroup take the steps of its segment (32 keys each) in
// turn, each with a maximum, sum and O of its own, and join them through LDS at the segment's end: no barrier
// inside the walk over the keys.
//   S^T (32 keys x 16 queries) = K . Q^T   v_mfma 16x16x32, A = K as loaded (lane: key l % 16, 16 bytes), B = Q^T
//   O^T (D x 16 queries) += V^T . P^T      A = V^T by transposing reads of the wave's own V rows in LDS
// S^T leaves lane l with queries l % 16 and keys 4 (l / 16) + r of both halves of the step, which are the
// k-slots of P^T once V^T is read in that order, so P^T goes from registers to the product.
// 8-bit rows are widened to 16 bits (exact) on their way; a key's scale multiplies its scores, a value's scale
// its P before the one rounding of P to the type: the operand of a 16-bit product, half a step of each weight (in 32 bits
// the product would be the fp32 matrix core's, a sixteenth of the rate). Scores, maxima, sums and O are fp32; the sum takes
// P before its rounding. Errors of the results against 64 bits, beside those of a form that holds P in fp32 too: bf16
// 0.0017 to 0.0018 of their size and 0.0017, fp16 0.00023 to 0.00024 and 0.00021.
// A value that is not finite must reach the rows that see it and no others, and 0 x infinity would be a NaN:
// a step that has one takes its P.V product in fp32 over the visible pairs instead.
// 64 single tokens over up to 8192 keys, 32 heads over 8, D = 128, bf16: 215 us, 5.5 TB/s; 32 over 16384, 32 over 4,
// e4m3: 60 us, 5.0 TB/s of codes and scales. One over 1031, which is latency: 9.8 us and 4.5 of the join.
//
// Workgroups on a CU: two, but for two blocks of 128 dims in 16 bits, whose queries (32 registers), O (64) and rows
// on their way (64) leave too few of half the registers (64 x 8 tokens over 8192 keys: 226 us, with two 260). One
// block with one, 16 bits, 256 x 1 over 700: 109 for 95; in 8 bits, 64 x 1 over 8192 and 64 dims, 108 for 81. Two blocks
// of 128 dims in 8 bits fit two workgroups with 16 (bf16) to 29 (fp16) registers in memory, and are faster than one
// workgroup without: 64 x 8 over 8192, int8, bf16 167 us and 187, fp16 185 and 194; e4m3, fp16 158 and 185.
constexpr int few_wgs(int d, bool k8, int nb) { return d == 128 && !k8 && nb == 2 ? 1 : 2; }
template <typename T, typename C, int D, int NB>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_wgs(D, cache_type<C>::k8bit, NB))))
paged_attn_few(PagedCache c, RowsQ a, AttnWork w) {
  typedef typename vec8<T>::type V8;
  constexpr bool k8 = cache_type<C>::k8bit;
  constexpr bool kUnits = k8 && std::is_same<T, f16>::value;      // each row's O in a unit of its own
  constexpr int WAVES = 4, ROWS = 16 * NB, RB = D * 2;            // RB: bytes of a V row in LDS
  constexpr int CB = k8 ? D : 2 * D;                              // bytes of a cache row
  constexpr int LPR = CB / 16, RPL = kWave / LPR, VL = kStep / RPL;   // V loads: lanes per row, rows per load, loads
  constexpr int KK = D / 32;                                      // 32-dim steps of a key block
  constexpr int KL = k8 ? D / 64 : KK;                            // K loads of a 16-key block
  constexpr int CR = D / 8;                                       // 16-byte chunks of a V row in LDS
  constexpr int NDB = D / 16;                                     // 16-dim blocks of O^T
  constexpr int WAVE_BYTES = kStep * RB;
  static_assert(WAVE_BYTES >= D * 16 * 4, "a wave's V rows make room for 16 rows of its O");
  __shared__ __attribute__((aligned(1024))) unsigned char v_lds[WAVES][WAVE_BYTES];
  __shared__ float stat_lds[WAVES][2][16];
  __shared__ float scale_lds[WAVES][2][kStep];
  __shared__ int64_t walk_lds[10];
  int tid = (int)threadIdx.x, lane = tid % kWave, g = lane / 16, lq = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // What follows from the lane (addresses, indexes of lanes, comparisons) is computed where it is used, in a few
  // instructions: hoisted out of the loops it costs 30 to 60 registers, which then go to memory.
  auto here = [&] { asm volatile("" : "+v"(tid), "+v"(lane), "+v"(g), "+v"(lq)); };

  PartRecord rec = {0, 0, 0, 0};
  WorkWalk walk;
  int wg;
  const bool active = start_walk<256>(c, w, false, walk_lds, wg, walk);
  Segment sg;
  unsigned char* vw = v_lds[wave];
  // Swizzled 16-byte chunk of a V row: the 8 rows x 2 chunks that 32 lanes of a transposing read touch lie in
  // distinct banks.
  auto v_at = [](int row, int chunk) {
    return row * RB + ((chunk ^ (CR == 16 ? 2 * (row & 7) : 2 * ((row >> 1) & 3))) * 16);
  };

  // Its reads and writes by lane: one base each, the rest by constants. A write of load i is i RPL rows below the
  // lane's first, whose swizzle differs where loads alternate between the halves of 8 rows.
  const int w_row = lane / LPR, w_chunk = lane % LPR * (k8 ? 2 : 1);
  int w_base = v_at(w_row, w_chunk), r_base = v_at(4 * g + lq / 4, lq % 4 / 2) + 8 * (lq % 2);
  auto v_write = [&](int i) { return i * RPL * RB + (w_base ^ (RPL == 4 && CR == 16 && i % 2 ? 128 : 0)); };

  InTile in_row[NB], out_row[NB];   // of the lane's columns, and of the rows that the thread joins
#pragma unroll
  for (int b = 0; b < NB; ++b) in_row[b] = in_tile(w.tiles, 16 * b + lq), out_row[b] = in_tile(w.tiles, 16 * b + tid / 16);
  while (active && uniform((int)walk.next([&](int s) { return uniform(load_seq(c, s)); }, sg)) != 0) {
    sg = {uniform(sg.rows), uniform(sg.seq), uniform(sg.head), uniform(sg.tile), uniform(sg.from), uniform(sg.to), uniform(sg.steps)};
    int kv_head, head_part;
    split_head(w.tiles, sg.head, kv_head, head_part);
    here();
    // ---- the tile's queries
    u32x4 qf[NB][KK];
    int seen[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      int token, hq;
      const bool mine = tile_row(w.tiles, sg.rows, sg.head, sg.tile, in_row[b], token, hq);
      seen[b] = mine ? keys_seen(sg.rows, token, c.capacity, w.causal) : 0;
      const T* qp = static_cast<const T*>(a.q) + (mine ? (int64_t)(sg.rows.first + token) * a.q_token + hq * a.q_head : 0);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int dim = k8 ? 64 * (kk / 2) + 16 * g + 8 * (kk % 2) : 32 * kk + 8 * g;
        qf[b][kk] = mine ? *reinterpret_cast<const u32x4*>(qp + dim) : u32x4{0, 0, 0, 0};
      }
    }
    int all_seen = seen[0], any_seen = seen[0];   // keys that every row, and that some row, sees
    {
      // (rows of no token count for neither)
      int lo = INT32_MAX, hi = 0;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        int token, hq;
        if (tile_row(w.tiles, sg.rows, sg.head, sg.tile, in_row[b], token, hq)) lo = min(lo, seen[b]), hi = max(hi, seen[b]);
      }
#pragma unroll
      for (int d = 1; d < 16; d *= 2) lo = min(lo, __shfl_xor(lo, d)), hi = max(hi, __shfl_xor(hi, d));
      all_seen = __builtin_amdgcn_readfirstlane(lo);
      any_seen = __builtin_amdgcn_readfirstlane(hi);
    }
    float m[NB], l[NB], unit[NB];
    f32x4 o[NB][NDB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b] = -INFINITY;
      l[b] = 0.f;
      unit[b] = kUnits ? kUnitLeast : 1.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[b][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // ---- loads of a step: each lane looks up one key (lane % 32), the others get it by lane. A step's page
    // table entries are loaded a step before its rows are, and looked at (find_row) when they are needed.
    u32x4 kr[2][KL], vr[VL];
    float ks = 0.f, vs = 0.f;
    const int* table = c.table + sg.seq * c.table_stride;
    const uint32_t page_rows = c.heads * c.page_size;
    auto load_page = [&](int step) { return table[page_of((uint32_t)min(step * kStep + lane % 32, c.capacity - 1), c.div)]; };
    auto find_row = [&](int step, int page) {
      const int key = step * kStep + lane % 32;
      const uint32_t at = (uint32_t)page * page_rows + kv_head * c.page_size + (key - page_of((uint32_t)key, c.div) * c.page_size);
      return key < any_seen && (unsigned)page < (unsigned)c.pages ? (int)at : -1;
    };
    auto load_step = [&](int row) {
      const int at = max(row, 0);   // (an absent row reads the cache's first one, and counts for nothing)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const unsigned char* p = static_cast<const unsigned char*>(c.k) + (int64_t)__shfl(at, 16 * b + lq) * CB;
#pragma unroll
        for (int i = 0; i < KL; ++i) kr[b][i] = *reinterpret_cast<const u32x4*>(p + 64 * i + 16 * g);
      }
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const unsigned char* p = static_cast<const unsigned char*>(c.v) + (int64_t)__shfl(at, i * RPL + lane / LPR) * CB;
        vr[i] = *reinterpret_cast<const u32x4*>(p + lane % LPR * 16);
      }
      if constexpr (k8) ks = c.k_scale[at], vs = c.v_scale[at];
    };

    int step = sg.from + wave, row = -1, page = 0;
    if (step < sg.to) {
      page = load_page(step);
      row = find_row(step, page);
      page = load_page(step + WAVES);
      load_step(row);
    }
    for (; step < sg.to; step += WAVES) {
      const unsigned present = (unsigned)__builtin_amdgcn_ballot_w64(row >= 0);   // of the step's 32 keys
      const int key0 = step * kStep;
      const bool clean = present == 0xffffffffu && key0 + kStep <= all_seen;
      // ---- V to LDS, S^T
      u16x2 top = {0, 0};
      here();
      if constexpr (k8) {   // (widened here, not before, where it would take twice the registers)
#pragma unroll
        for (int i = 0; i < VL; ++i) asm volatile("" : "+v"(vr[i]));
#pragma unroll
        for (int i = 0; i < KL; ++i) asm volatile("" : "+v"(kr[0][i]), "+v"(kr[1][i]));
      }
      asm volatile("" : "+v"(w_base), "+v"(r_base));
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int r = i * RPL + lane / LPR;
        if (present != 0xffffffffu && !(present >> r & 1)) vr[i] = u32x4{0, 0, 0, 0};
        if constexpr (k8) {
          u32x4 x, y;
          widen16<C, T>(vr[i], x, y);
          top = max_bits(max_bits(top, x), y);
          *reinterpret_cast<u32x4*>(vw + v_write(i)) = x;
          *reinterpret_cast<u32x4*>(vw + (v_write(i) ^ 16)) = y;
        } else {
          top = max_bits(top, vr[i]);
          *reinterpret_cast<u32x4*>(vw + v_write(i)) = vr[i];
        }
      }
      const bool odd = __builtin_amdgcn_ballot_w64(max(top[0], top[1]) >= kInfBits<T>) != 0;
      f32x4 s[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) s[b][0] = s[b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          u32x4 x, y;
          if constexpr (k8) {
            widen16<C, T>(kr[h][kk / 2], x, y);
            if (kk % 2) x = y;
          } else {
            x = kr[h][kk];
          }
#pragma unroll
          for (int b = 0; b < NB; ++b)
            s[b][h] = mfma16x16x32(__builtin_bit_cast(V8, x), __builtin_bit_cast(V8, qf[b][kk]), s[b][h]);
        }
      f32x4 ksc[2], vsc[2];
      if constexpr (k8) {
        if (lane < 32) scale_lds[wave][0][lane] = ks, scale_lds[wave][1][lane] = vs;
      }
      // ---- the next step's rows, into the registers that this one's have left
      __builtin_amdgcn_sched_barrier(0);
      if (step + WAVES < sg.to) {
        row = find_row(step + WAVES, page);
        page = load_page(step + 2 * WAVES);
        load_step(row);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (k8) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ksc[h] = *reinterpret_cast<const f32x4*>(&scale_lds[wave][0][16 * h + 4 * g]) * w.scale_log2;
          vsc[h] = *reinterpret_cast<const f32x4*>(&scale_lds[wave][1][16 * h + 4 * g]);
        }
      }
      // ---- softmax
      V8 pf[NB];
      float p32[NB][8];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float t[8];
        // Keys (of this lane, j = 4 half + r) that the row sees: bit j.
        unsigned sees = 0xff;
        float mx = kLowest;   // (lowered in the branch: behind it, 64 x 8 tokens over an int8 cache take 313 us for 275)
        if (!clean) {
          sees = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int k = 16 * (j / 4) + 4 * g + j % 4;
            sees |= key0 + k < seen[b] && (present >> k & 1) ? 1u << j : 0u;
          }
          mx = sees ? kLowest : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          t[j] = s[b][j / 4][j % 4] * (k8 ? ksc[j / 4][j % 4] : w.scale_log2);
          if (!clean) t[j] = sees >> j & 1 ? t[j] : -INFINITY;
          mx = fmaxf(mx, t[j]);
        }
        const float m_new = fmaxf(m[b], groups_max(mx));
        const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
        if (__builtin_amdgcn_ballot_w64(m_new > m[b]) != 0) {
          const float f = m[b] == -INFINITY ? 0.f : exp2_fast(m[b] + neg_m);
          l[b] *= f;
          if constexpr (kUnits) {
            unit[b] *= f;
          } else {
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[b][db] *= f;
          }
          m[b] = m_new;
        }
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float p = exp2_fast(t[j] + neg_m);
          l[b] += p;
          if constexpr (k8) {
            p *= vsc[j / 4][j % 4];
            if (!clean) p = sees >> j & 1 ? p : 0.f;   // (0 x a scale that is not finite)
          }
          if constexpr (kUnits) top = fmaxf(top, fabsf(p));
          p32[b][j] = p;
        }
        if constexpr (kUnits) {
          const float was = unit[b], now = unit_for(fmaxf(was, kUnitLeast), groups_max(top));
          if (__builtin_amdgcn_ballot_w64(now != was) != 0) {
            const float f = now == was ? 1.f : was / now;
            unit[b] = now;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[b][db] *= f;
          }
          const float inv = __builtin_amdgcn_rcpf(now);
#pragma unroll
          for (int j = 0; j < 8; ++j) p32[b][j] *= inv;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[b][j] = from_f32<T>(p32[b][j]);
      }
      // ---- O^T += V^T . P^T
      if (!odd) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const unsigned char* p = vw + (r_base ^ (32 * db));
          const i16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p));
          const i16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p + 16 * RB));
          const i16x8 x = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
#pragma unroll
          for (int b = 0; b < NB; ++b) o[b][db] = mfma16x16x32(__builtin_bit_cast(V8, x), pf[b], o[b][db]);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < kStep; ++k) {
          here();
          const int from = (k % 16) / 4 * 16 + lq, j = k / 16 * 4 + k % 4;
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) p = i == j ? p32[b][i] : p;
            p = __shfl(p, from);
            if (key0 + k < seen[b] && (present >> k & 1)) {
#pragma unroll
              for (int db = 0; db < NDB; ++db) {
                typedef T T4 __attribute__((ext_vector_type(4)));
                const T4 x = *reinterpret_cast<const T4*>(vw + v_at(k, 2 * db + g / 2) + 8 * (g % 2));
#pragma unroll
                for (int r = 0; r < 4; ++r) o[b][db][r] = fmaf(p, to_f32(x[r]), o[b][db][r]);
              }
            }
          }
        }
      }
    }

    // ---- join the waves, 16 rows at a time through the V rows' LDS
    const bool done = sg.from == 0 && sg.to == sg.steps;
    const int slot = sg.from == 0 ? 1 : 0;
    if (!done) {
      if (sg.from == 0) rec = {sg.seq, sg.head, sg.tile, rec.flags | kPartBegins};
      else rec.flags |= kPartContinues | (sg.to == sg.steps ? kPartEnds : 0);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      here();
      const float ls = groups_sum(l[b]);
#pragma unroll
      for (int db = 0; db < NDB; ++db)
        *reinterpret_cast<f32x4*>(vw + lq * (D * 4) + (((4 * db + g) ^ lq) * 16)) = o[b][db] * unit[b];
      if (lane < 16) stat_lds[wave][0][lane] = m[b], stat_lds[wave][1][lane] = ls;
      __syncthreads();
      const int q = tid / 16, part = tid % 16;   // 16 threads a row, D / 16 dims each
      constexpr int EL = D / 16;
      float mx = -INFINITY, sum = 0.f, x[EL] = {};
#pragma unroll
      for (int i = 0; i < WAVES; ++i) mx = fmaxf(mx, stat_lds[i][0][q]);
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        const float f = stat_lds[i][0][q] == -INFINITY ? 0.f : exp2_fast(stat_lds[i][0][q] - mx);
        sum = fmaf(f, stat_lds[i][1][q], sum);
#pragma unroll
        for (int e = 0; e < EL; e += 4) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(&v_lds[i][q * (D * 4) + (((part * (EL / 4) + e / 4) ^ q) * 16)]);
          if (f > 0.f)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[e + j] = fmaf(f, y[j], x[e + j]);
        }
      }
      int token, hq;
      if (tile_row(w.tiles, sg.rows, sg.head, sg.tile, out_row[b], token, hq)) {
        if (done) {
          typedef T TE __attribute__((ext_vector_type(EL)));
          TE y;
#pragma unroll
          for (int e = 0; e < EL; ++e) y[e] = from_f32<T>(row_result(x[e], mx, sum));
          *reinterpret_cast<TE*>(static_cast<T*>(a.o) + (int64_t)(sg.rows.first + token) * a.o_token + hq * a.o_head + part * EL) = y;
        } else {
          float* to = part_rows(w, wg, slot, ROWS, D) + (16 * b + q) * D + part * EL;
#pragma unroll
          for (int e = 0; e < EL; e += 4) *reinterpret_cast<f32x4*>(to + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
          if (part == 0) {
            float* st = part_stats(w, (int)gridDim.x, wg, slot, ROWS, D);
            st[16 * b + q] = mx, st[ROWS + 16 * b + q] = sum;
          }
        }
      }
      __syncthreads();
    }
  }
  if (tid == 0) w.records[wg] = rec;
}

// ---- Many rows a tile: chunks of prompts ----
//
// A tile has BM rows, 32 for each wave; its keys go past in tiles of 64 that all waves share in LDS: 4 D x 64 x BM
// operations for 4 D x 64 bytes (2 D in 8 bits), so that the matrix core bounds the kernel, and beside it the
// exponentials. Both products as in fa_mfma.hpp, transposed on 32x32x16 MFMAs with a query per lane, in two stages
// that overlap: the matrix core takes S(t+1) beside half of the exponentials of P(t), and O += V(t) P(t) beside half
// of those of P(t+1). K(t+2) and V(t+1) arrive meanwhile, a row per page lookup: 16-bit rows straight into LDS;
// 8-bit rows into a raw buffer of LDS one tile earlier, each thread its own, and from there widened to 16 bits
// (exact) once for all waves. A key's scale multiplies its scores, a value's scale its P before the one rounding of
// P to the type (fp16: in the row's unit), an operand in 16 bits as in the kernel above; in 16 bits the sum takes the
// rounded P, two weights an instruction, so that numerator and sum are of the same weights. Errors
// as above: bf16 over e4m3 0.0023 and 0.0017, bf16 0.0019 and 0.0017, fp16 0.00025 and 0.00020.
// O and l are rescaled only when some row's maximum outgrew its reference by more than 2^8.
// A value that is not finite must not reach rows that do not see it (0 x infinity is NaN): of a tile that some row
// does not see whole, each wave looks at its share of the values as they arrive; if one is not finite, the pipeline
// ends there. The tiles from it on go one by one, those with such a value leave P . V out, and it is added at the
// end in fp32 over the visible pairs.
// 4096 tokens at the end of 32768 keys, 32 heads over 8, D = 128, causal: bf16 1.93 to 2.09 ms, 990 to 1070
// TFLOP/s (the card's large matrix products reach 1290), fp16 2.03 to 2.07; e4m3 and int8 with bf16 2.24 and 2.33 ms, with
// fp16, whose units cost three more VALU operations a pair of scores and 9 to 16 registers in memory, 2.51 and 2.58; D = 64
// 1.28 ms, int8 1.75, with fp16 2.04.
//
// Rows of a tile, D = 128, 256 and 128 (one workgroup of 8 waves on a CU, two of 4): that case 2015 and 2183 us, 4 x
// 2048 120 and 117, 24 x 700 over 4096 456 and 491, 256 x 64 over 640 73 and 85. D = 64 has 128, and as many
// workgroups on a CU as the registers allow, three in 16 bits (4 x 2048 tokens f16 88 us, with two 100), two in 8
// (with three 24 x 700 over 4096 in int8 takes 493 for 480).
constexpr int chunk_rows_of(int d) { return d == 128 ? 256 : 128; }
constexpr int chunk_wgs(int d, bool k8) { return d == 128 ? 1 : k8 ? 2 : 3; }   // workgroups on a CU

// WIDE: caches (or their scales) past a buffer's 32-bit offsets. 16-bit rows then come from 64-bit addresses by
// instructions of the flat kind, after which the compiler waits for all LDS reads instead of the oldest; 8-bit ones
// are not pipelined at all. The case above takes 2108 us (in buffers 1976), in int8 3129 (2312), with D = 64 2659 (1756).
constexpr uint32_t kPastBuffer = 0xffffe000u;
template <typename T, typename C, int D, int BM, bool WIDE>
__global__ void __launch_bounds__(BM * 2) __attribute__((amdgpu_waves_per_eu(chunk_wgs(D, cache_type<C>::k8bit) * BM / 128)))
paged_attn_chunk(PagedCache c, RowsQ a, AttnWork w) {
  typedef typename vec8<T>::type V8;
  constexpr bool k8 = cache_type<C>::k8bit;
  constexpr bool kUnits = k8 && std::is_same<T, f16>::value;   // each row's O in a unit of its own
  constexpr int BN = 64, THREADS = BM * 2, RB = D * 2, CB = k8 ? D : 2 * D, CR = D / 8;
  constexpr int TILE_BYTES = BN * RB;
  constexpr int QK_STEPS = D / 16, NKB = BN / 32, NDB = D / 32, PV_STEPS = BN / 16;
  constexpr int CPT = BN * CB / 16 / THREADS;   // 16-byte loads per thread, matrix and tile
  constexpr int LPR = CB / 16;                  // lanes a cache row
  static_assert(CPT * THREADS * 16 == BN * CB, "a tile's loads split evenly");
  constexpr float kLazyLog2 = 8.f;
  __shared__ __attribute__((aligned(1024))) unsigned char k_lds0[TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char v_lds0[TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char k_lds1[TILE_BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char v_lds1[TILE_BYTES];
  // 8 bits: rows as they are, each thread's own, on their way to the stages; and four tiles' scales.
  constexpr int RAW = k8 && !WIDE ? BN * CB : 16, SLOTS = k8 ? 4 : 1;
  __shared__ __attribute__((aligned(1024))) unsigned char k_raw0[RAW], k_raw1[RAW], v_raw0[RAW], v_raw1[RAW];
  __shared__ __attribute__((aligned(256))) float ks_lds[SLOTS][BN], vs_lds[SLOTS][BN];
  __shared__ float ones_lds[k8 ? BN : 1];
  __shared__ int odd_lds[2][BM / 32];   // of V(t), at t % 2: whether a wave's share has a value that is not finite
  __shared__ int64_t walk_lds[10];
  const std::integral_constant<int, 0> even{};
  const std::integral_constant<int, 1> odd{};
  auto k_stage = [&](auto par) -> unsigned char* { if constexpr (decltype(par)::value) return k_lds1; else return k_lds0; };
  auto v_stage = [&](auto par) -> unsigned char* { if constexpr (decltype(par)::value) return v_lds1; else return v_lds0; };
  const int tid = (int)threadIdx.x, wave = uniform(tid / kWave), lane = tid % kWave;
  const int lq = lane % 32, hi = lane / 32, g16 = lane / 16, i16 = lane % 16;

  // Operand read addresses (fa_mfma.hpp): K row lq, chunk 2 kk + hi; V^T by transposing reads.
  // The swizzles reach chunk bits that the step and the dim block do not, so those enter by XOR.
  const int v_row = hi * 4 + i16 / 4, v_cl = 2 * (g16 % 2) + (i16 % 4) / 2;
  int k_base = lq * RB + ((hi ^ k_swz<CR>(lq)) * 16), v_base = v_row * RB + ((v_cl ^ v_swz<CR>(v_row)) * 16) + 8 * (i16 % 2);
  const uint32_t cache_bytes = (uint32_t)min((uint64_t)c.pages * c.heads * c.page_size * CB, (uint64_t)kPastBuffer);
  const rsrc_t k_rs = make_rsrc(c.k, cache_bytes), v_rs = make_rsrc(c.v, cache_bytes);
  const uint32_t scale_bytes = k8 ? (uint32_t)min((uint64_t)c.pages * c.heads * c.page_size * 4, (uint64_t)kPastBuffer) : 0;
  const rsrc_t ks_rs = make_rsrc(k8 ? c.k_scale : nullptr, scale_bytes), vs_rs = make_rsrc(k8 ? c.v_scale : nullptr, scale_bytes);

  if (k8 && tid < BN) ones_lds[tid] = 1.f;   // (before the barriers of start_walk)
  PartRecord rec = {0, 0, 0, 0};
  WorkWalk walk;
  int wg;
  const bool active = start_walk<THREADS>(c, w, true, walk_lds, wg, walk);
  Segment sg;
  const InTile in_row = in_tile(w.tiles, 32 * wave + lq);
  constexpr int AHEAD = k8 ? 3 : 2;
  int kv_head, key_begin, key_end, wave_all, wave_any;
  int pages[AHEAD + 1], page, in_page;   // in_page: the row in its page of the key whose entry `page` is
  V8 qf[QK_STEPS];
  // The lane's row. Found again for each use, not held over the loops.
  int token, hq, seen;
  bool mine;
  auto find_mine = [&]() {
    InTile r = in_row;
    asm volatile("" : "+v"(r.token), "+v"(r.head));
    mine = tile_row(w.tiles, sg.rows, sg.head, sg.tile, r, token, hq);
    seen = mine ? keys_seen(sg.rows, token, c.capacity, w.causal) : 0;
  };
  auto load_page = [&](int t, int& rest) {
    const int pos = min(key_begin + t * BN + lane, c.capacity - 1);
    const int col = (int)page_of((uint32_t)pos, c.div);
    rest = pos - col * c.page_size;
    return c.table[sg.seq * c.table_stride + col];
  };
  auto in_page_of = [&](int t) {
    const int key = key_begin + t * BN + lane;
    return key - (int)page_of((uint32_t)key, c.div) * c.page_size;
  };
  // The next segment: its queries and first page table entries on their way. (Called before the stores of the one
  // before it, which they need not wait for.)
  auto begin_segment = [&]() __attribute__((always_inline)) {
    if (uniform((int)walk.next([&](int s) { return uniform(load_seq(c, s)); }, sg)) == 0) return false;
    sg = {uniform(sg.rows), uniform(sg.seq), uniform(sg.head), uniform(sg.tile), uniform(sg.from), uniform(sg.to), uniform(sg.steps)};
    int head_part;
    split_head(w.tiles, sg.head, kv_head, head_part);
    // Keys of the segment's tile: up to the last row's.
    const int last_token = min((sg.tile + 1) * w.tiles.tokens, sg.rows.count) - 1;
    key_begin = sg.from * kStep;
    key_end = min(sg.to * kStep, keys_seen(sg.rows, last_token, c.capacity, w.causal));
#pragma unroll
    for (int j = 0; j <= AHEAD; ++j) pages[j] = load_page(j, in_page);
    page = load_page(AHEAD + 1, in_page);
    find_mine();
    const T* qp = static_cast<const T*>(a.q) + (mine ? (int64_t)(sg.rows.first + token) * a.q_token + hq * a.q_head : 0) + 8 * hi;
#pragma unroll
    for (int kk = 0; kk < QK_STEPS; ++kk) {
      const u32x4 x = mine ? *reinterpret_cast<const u32x4*>(qp + 16 * kk) : u32x4{0, 0, 0, 0};
      qf[kk] = __builtin_bit_cast(V8, x);
    }
    // Keys that all of the wave's rows see, and that some row does (none: the wave has no rows).
    int lo = mine ? seen : INT32_MAX, up = seen;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) lo = min(lo, __shfl_xor(lo, d)), up = max(up, __shfl_xor(up, d));
    wave_all = uniform(lo), wave_any = uniform(up);
    return true;
  };
  bool more = active && begin_segment();
  while (more) {
    const int nt = max(1, (key_end - key_begin + BN - 1) / BN);

    // ---- tiles of keys: lane l looks up key l; each thread's chunk rows come from there by lane
    const uint32_t page_rows = c.heads * c.page_size, head_rows = kv_head * c.page_size;
    auto find_row = [&](int t, int page, int rest) {
      const int key = key_begin + t * BN + lane;
      const uint32_t at = (uint32_t)page * page_rows + (head_rows + rest);
      const bool there = (key < key_end) & ((unsigned)page < (unsigned)c.pages);
      return there ? (int)at : -1;
    };
    // 16-bit rows: thread's load i fills LDS slot i THREADS + tid, which holds the swizzled chunk of its row (loads
    // are 32 rows apart, so the swizzle is the same).
    static_assert(k8 || THREADS / LPR == 32, "loads 32 rows apart");
    const int k_off = (tid % LPR ^ k_swz<CR>(tid / LPR)) * 16, v_off = (tid % LPR ^ v_swz<CR>(tid / LPR)) * 16;
    auto to_lds = [&](const void* cache, rsrc_t rs, const int (&rows)[CPT], unsigned char* stage, bool is_v) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        unsigned off = is_v ? v_off : k_off;
        asm("" : "+v"(off));   // (not to be added to the base once for all loads: that spills)
        unsigned char* to = stage + (i * THREADS + wave * kWave) * 16;
        if constexpr (WIDE) {
          const unsigned char* p = static_cast<const unsigned char*>(cache) + ((uint64_t)(unsigned)rows[i] * CB + off);
          __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
        } else {
          load16_to_lds(rs, to, (unsigned)rows[i] + off, 0);
        }
      }
    };
    // 8-bit rows: through registers, or into the thread's 16 bytes of a raw buffer; then widened and stored.
    static_assert(!k8 || CPT == 1, "one load of 8-bit rows a thread");
    auto to_regs = [&](const void* cache, rsrc_t rs, const int (&rows)[CPT], u32x4 (&x)[CPT]) {
      if constexpr (WIDE) x[0] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(cache) + (uint64_t)(unsigned)rows[0] * CB + tid % LPR * 16);
      else x[0] = load16(rs, (unsigned)rows[0] + tid % LPR * 16);
    };
    auto to_raw = [&](rsrc_t rs, const int (&rows)[CPT], unsigned char* raw) {
      load16_to_lds(rs, raw + wave * kWave * 16, (unsigned)rows[0] + tid % LPR * 16, 0);
    };
    auto from_raw = [&](const unsigned char* raw, u32x4 (&x)[CPT]) { x[0] = *reinterpret_cast<const u32x4*>(raw + tid * 16); };
    auto widen = [&](const u32x4 (&x)[CPT], unsigned char* stage, bool is_v) {
      if constexpr (k8) {
        int at = tid;
        asm("" : "+v"(at));   // (addresses made each time, not held)
        const int r = at / LPR, ch = (at % LPR * 2) ^ (is_v ? v_swz<CR>(r) : k_swz<CR>(r));
        u32x4 lo16, hi16;
        widen16<C, T>(x[0], lo16, hi16);
        *reinterpret_cast<u32x4*>(stage + r * RB + ch * 16) = lo16;
        *reinterpret_cast<u32x4*>(stage + r * RB + (ch ^ 1) * 16) = hi16;
      }
    };
    auto present_of = [&](int row) -> uint64_t { return __builtin_amdgcn_ballot_w64(row >= 0); };
    // The row that each of the thread's loads reads; where loads are from a buffer, its byte offset, past the
    // buffer's end (which loads as zeros) for an absent key. Elsewhere an absent key takes the row of the tile's
    // first present one: its scores are masked, and its P is 0, which a finite value leaves without effect.
    auto chunk_rows = [&](int row, uint64_t pres, int (&rows)[CPT]) {
      if constexpr (WIDE) {
        const int first = max(__builtin_amdgcn_readlane(row, __builtin_ctzll(pres | 1ull << 63)), 0);
        row = row < 0 ? first : row;
      } else {
        row = row < 0 ? (int)kPastBuffer : (int)((unsigned)row * CB);
      }
#pragma unroll
      for (int i = 0; i < CPT; ++i) rows[i] = __shfl(row, (i * THREADS + tid) / LPR);
    };
    // A tile's scales by lane = key, into its slot: wave 0 the keys', wave 1 the values'. Absent keys get zeros.
    auto load_scale = [&](int row) {
      const float x = wave < 2 && row >= 0 ? (wave ? c.v_scale : c.k_scale)[row] : 0.f;
      return x;
    };
    auto store_scale = [&](int t, float x) {
      if (wave < 2) (wave ? vs_lds : ks_lds)[t % SLOTS][lane] = x;
    };
    auto scales_to_lds = [&](int t, int row) {   // (4 bytes a lane)
      if (wave < 2)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wave ? vs_rs : ks_rs, (__attribute__((address_space(3))) void*)&(wave ? vs_lds : ks_lds)[t % SLOTS][0],
                                                 4, row < 0 ? kPastBuffer : (unsigned)row * 4, 0, 0, 0);
    };
    // The wave's first tile that is not clean and has a value that is not finite: from there on, tiles that are
    // not clean leave P . V out, and take_visible adds it at the end.
    int skip_from = INT32_MAX;
    float m_run = -INFINITY, unit = kUnits ? kUnitLeast : 1.f, l = 0.f;
    f32x16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] = f32x16{};

    // (The operands' addresses are made from their base each time: hoisted out of the loops, they spill.)
    auto qk = [&](f32x16 (&s)[NKB], const unsigned char* ks) {
      int kb = k_base;
      asm("" : "+v"(kb));
#pragma unroll
      for (int b = 0; b < NKB; ++b) s[b] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < QK_STEPS; ++kk)
#pragma unroll
        for (int b = 0; b < NKB; ++b)
          s[b] = mfma32x32x16(*reinterpret_cast<const V8*>(ks + b * 32 * RB + (kb ^ (32 * kk))), qf[kk], s[b]);
    };
    // Keys' scales.
    auto scale_scores = [&](f32x16 (&s)[NKB], int t) {
      if constexpr (k8)
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(&ks_lds[t % SLOTS][32 * b + 8 * q4 + 4 * hi]);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[b][4 * q4 + r] *= x[r];
          }
    };
    // Keys of a tile that this lane's row sees, as bits: 32-key block b, bit 8 (r / 4) + r % 4 for the key of
    // register r (the lane's keys begin 4 hi further on).
    struct Bits { unsigned b[NKB]; };
    auto visible = [&](int t, uint64_t present) {
      Bits v;
#pragma unroll
      for (int b = 0; b < NKB; ++b) {
        const int n = clamp_int(seen - (key_begin + t * BN + 32 * b), 0, 32);
        const unsigned below = n == 32 ? ~0u : (1u << n) - 1;
        v.b[b] = ((unsigned)(present >> (32 * b)) & below) >> (4 * hi);
      }
      return v;
    };
    auto mask = [&](f32x16 (&s)[NKB], int t, uint64_t present) {   // gives the least of the maximum
      const Bits v = visible(t, present);
      constexpr unsigned kMine = 0x0f0f0f0fu;   // the lane's keys
      unsigned any = 0;
#pragma unroll
      for (int b = 0; b < NKB; ++b) {
        any |= v.b[b] & kMine;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = v.b[b] & 1u << (8 * (r / 4) + r % 4) ? s[b][r] : -INFINITY;
      }
      return any ? kLowest : -INFINITY;
    };
    auto row_max = [&](const f32x16 (&s)[NKB], float mx) {
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int r = 0; r < 16; r += 2) mx = max_nan(mx, max_nan(s[b][r], s[b][r + 1]));
      return max_nan(mx, partner32(mx)) * w.scale_log2;
    };
    auto raise = [&](float mx) {   // the reference maximum, where some row's grew past 2^8: whether it did
      const float m_new = fmaxf(m_run, mx);
      const bool up = __builtin_amdgcn_ballot_w64(m_new > m_run + kLazyLog2) != 0;
      if (up) {
        const float f = m_new > m_run ? exp2_fast(m_run - m_new) : 1.f;   // (m_run = -inf: 0)
        m_run = m_new;
        l *= f;
        float g = f;
        if constexpr (kUnits) {   // (the unit falls instead of O, down to its least)
          const float to = fmaxf(unit * f, kUnitLeast);
          g = unit * f == to ? 1.f : unit * f / to;
          unit = to;
        }
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] *= g;
      }
      return up;
    };
    auto exponentiate = [&](const f32x16 (&s)[NKB], V8 (&pf)[PV_STEPS]) {
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) pf[b * 2 + r / 8][r % 8] = from_f32<T>(exp2_fast(fmaf(s[b][r], w.scale_log2, neg_m)));
    };
    // 8 bits: the sum takes P, the product P times the values' scales (in fp16 in the row's unit; `top` takes the largest).
    // (The product with a scale takes 0 for a P of 0 whatever the scale: of a key that the row does not see, it may
    // not be finite.)
    auto exponentiate8 = [&](const f32x16 (&s)[NKB], V8 (&pf)[PV_STEPS], int t, float& sum, float& top) __attribute__((always_inline)) {
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      const float inv = kUnits ? __builtin_amdgcn_rcpf(unit) : 1.f;
      sum = top = 0.f;
#pragma unroll
      for (int b = 0; b < NKB; ++b)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(&vs_lds[t % SLOTS][32 * b + 8 * q4 + 4 * hi]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float p = exp2_fast(fmaf(s[b][4 * q4 + r], w.scale_log2, neg_m));
            sum += p;
            p = p == 0.f ? 0.f : p * x[r];
            if constexpr (kUnits) top = fmaxf(top, fabsf(p)), p *= inv;
            pf[b * 2 + q4 / 2][(q4 % 2) * 4 + r] = from_f32<T>(p);
          }
        }
    };
    // The rows' units, for weights of up to `top` in the lane: whether some changed. scaled: what O was multiplied by.
    auto raise_units = [&](float top, float& scaled) {
      if constexpr (!kUnits) return false;
      const float was = unit, now = unit_for(was, fmaxf(top, partner32(top)));
      if (__builtin_amdgcn_ballot_w64(now != was) == 0) return false;
      scaled = now == was ? 1.f : was / now;
      unit = now;
#pragma unroll
      for (int db = 0; db < NDB; ++db) o[db] *= scaled;
      return true;
    };
    auto pv = [&](const V8 (&pf)[PV_STEPS], const unsigned char* vs) {
      int vb = v_base;
      asm("" : "+v"(vb));
#pragma unroll
      for (int i = 0; i < PV_STEPS; ++i)
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const unsigned char* p0 = vs + i * 16 * RB + (vb ^ (64 * db));
          const i16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p0));
          const i16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p0 + 8 * RB));
          const i16x8 x = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
          o[db] = mfma32x32x16(__builtin_bit_cast(V8, x), pf[i], o[db]);
        }
    };
    // l of the lane's keys from the rounded P, as the products take it. Not by a product with a constant operand: its
    // zeros would carry one row's NaN into another's sum.
    auto row_sum = [&](const V8 (&pf)[PV_STEPS]) {
#pragma unroll
      for (int i = 0; i < PV_STEPS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) l = add_pair(__builtin_bit_cast(u32x4, pf[i])[j], l, static_cast<T*>(nullptr));
    };
    // The wave's own share of V(t) in LDS, and its scales: whether all of it is finite, for all waves after the next
    // barrier.
    auto check_values = [&](int t, const unsigned char* vs) {
      constexpr int N = TILE_BYTES / 16 / THREADS;
      u16x2 top = {0, 0};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = k8 ? (wave * N + i) * kWave + lane : i * THREADS + tid;
        top = max_bits(top, *reinterpret_cast<const u32x4*>(vs + at * 16));
      }
      bool odd_here = max(top[0], top[1]) >= kInfBits<T>;
      if constexpr (k8) odd_here = odd_here || !(fabsf(vs_lds[t % SLOTS][lane]) < INFINITY);
      const bool any = __builtin_amdgcn_ballot_w64(odd_here) != 0;
      if (lane == 0) odd_lds[t & 1][wave] = any;
    };
    auto values_finite = [&](int t) { return __builtin_amdgcn_ballot_w64(odd_lds[t & 1][lane % (BM / 32)] != 0) == 0; };
    const int wave_tiles = (min(wave_any, key_end) - key_begin + BN - 1) / BN;   // tiles with a key for some row of the wave
    auto is_clean = [&](int t, uint64_t pres) { return pres == ~0ull && key_begin + (t + 1) * BN <= wave_all; };

    // ---- the first tiles: K(0), V(0), K(1). At a tile t: rows[j] and row[j] are tile t + 1 + j's, present[j] tile
    // t + j's; page holds tile t + 1 + AHEAD's entries.
    int row[AHEAD], rows[AHEAD][CPT];
    uint64_t present[AHEAD + 1];
    const int tile_all = keys_seen(sg.rows, sg.tile * w.tiles.tokens, c.capacity, w.causal);   // the first row's keys
    auto whole_tile = [&](int t, uint64_t pres) { return pres == ~0ull && key_begin + (t + 1) * BN <= tile_all; };
    auto advance = [&](int next_row, uint64_t next_present) {   // to the next tile (its new rows[AHEAD - 1] apart)
#pragma unroll
      for (int j = 0; j + 1 < AHEAD; ++j) {
        row[j] = row[j + 1];
#pragma unroll
        for (int i = 0; i < CPT; ++i) rows[j][i] = rows[j + 1][i];
      }
      row[AHEAD - 1] = next_row;
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) present[j] = present[j + 1];
      present[AHEAD] = next_present;
    };
    {
      int row0, rows0[CPT];
      row0 = find_row(0, pages[0], in_page_of(0));
      present[0] = present_of(row0);
      chunk_rows(row0, present[0], rows0);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        row[j] = find_row(j + 1, pages[j + 1], in_page_of(j + 1));
        present[j + 1] = present_of(row[j]);
        chunk_rows(row[j], present[j + 1], rows[j]);
      }
      if constexpr (k8) {
        u32x4 kx[CPT], vx[CPT], k1[CPT];
        to_regs(c.k, k_rs, rows0, kx);
        to_regs(c.v, v_rs, rows0, vx);
        const float scale = load_scale(row0);
        if constexpr (!WIDE) {
          to_regs(c.k, k_rs, rows[0], k1);   // K(1), K(2) and V(1) too
          scales_to_lds(1, row[0]);
          to_raw(k_rs, rows[1], k_raw0);
          to_raw(v_rs, rows[0], v_raw1);
          widen(k1, k_stage(odd), false);
        }
        store_scale(0, scale);
        widen(kx, k_stage(even), false);
        widen(vx, v_stage(even), true);
      } else {
        to_lds(c.k, k_rs, rows0, k_stage(even), false);
        to_lds(c.v, v_rs, rows0, v_stage(even), true);
        to_lds(c.k, k_rs, rows[0], k_stage(odd), false);
      }
    }
    __builtin_amdgcn_s_waitcnt(0);
    if (!whole_tile(0, present[0])) {
      if (k8) __syncthreads();   // (the scales are waves 0 and 1's)
      check_values(0, v_lds0);
    }
    __syncthreads();
    // The pipeline takes a tile that every row sees whole, or that has finite values.
    auto fits = [&](int t, uint64_t pres) { return t < nt && (whole_tile(t, pres) || values_finite(t)); };

    // ---- the tiles in the two-stage pipeline
    int t0 = 0;   // tiles done
    if constexpr (!(k8 && WIDE)) {
      constexpr int HALF = PV_STEPS / 2;
      auto neg_ref = [&]() { return m_run == -INFINITY ? 0.f : -m_run; };
      // P of four scores, e to e + 3 (16-key step e / 8), of tile t; 8 bits: its sum to `sum`, in fp16 its largest weight
      // to `top`. (A masked score gives 0, and 0 times a scale is 0: a tile with a scale that is not finite and a masked
      // key does not come here.)
      auto exp_quad = [&](const f32x16 (&s)[NKB], V8 (&pf)[PV_STEPS], int e, float neg_m, int t, float inv, float& sum, float& top) __attribute__((always_inline)) {
        f32x4 x = {1.f, 1.f, 1.f, 1.f};
        if constexpr (k8) x = *reinterpret_cast<const f32x4*>(&vs_lds[t % SLOTS][e / 16 * 32 + e % 16 * 2 + 4 * hi]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float p = exp2_fast(fmaf(s[e / 16][e % 16 + k], w.scale_log2, neg_m));
          if constexpr (k8) {
            sum += p;
            p *= x[k];
            if constexpr (kUnits) top = max_nan(top, fabsf(p)), p *= inv;
          }
          pf[e / 8][e % 8 + k] = from_f32<T>(p);
        }
      };
      auto inverse_unit = [&]() { return kUnits ? __builtin_amdgcn_rcpf(unit) : 1.f; };
      float l_next = 0.f, top = 0.f;   // 8 bits: the sum of the first half of P(t + 1); its largest weight so far
      auto exp_first = [&](const f32x16 (&s)[NKB], V8 (&pf)[PV_STEPS], int t) __attribute__((always_inline)) {
        const float neg_m = neg_ref(), inv = inverse_unit();
        l_next = top = 0.f;
#pragma unroll
        for (int e = 0; e < HALF * 8; e += 4) exp_quad(s, pf, e, neg_m, t, inv, l_next, top);
      };
      // The first half of P(t) after its reference was raised (again) or its unit. (A second time at most: the unit then
      // has room for the same weights.)
      auto settle_first = [&](const f32x16 (&s)[NKB], V8 (&pf)[PV_STEPS], int t, bool again) __attribute__((always_inline)) {
        if constexpr (!kUnits) {
          if (again) exp_first(s, pf, t);
        } else {
          float scaled;
          do {
            if (again) exp_first(s, pf, t);
            again = raise_units(top, scaled);
          } while (again);
        }
      };
      f32x16 sa[NKB], sb[NKB];
      V8 pa[PV_STEPS], pb[PV_STEPS];
      if (fits(0, present[0])) {
        qk(sa, k_stage(even));
        scale_scores(sa, 0);
        raise(row_max(sa, is_clean(0, present[0]) ? kLowest : mask(sa, 0, present[0])));
        settle_first(sa, pa, 0, true);
        __syncthreads();   // iteration 0 replaces K(0)
        auto iteration = [&](auto par, int t, f32x16 (&s)[NKB], f32x16 (&sn)[NKB], V8 (&pf)[PV_STEPS], V8 (&pn)[PV_STEPS]) __attribute__((always_inline)) {
          constexpr int P = decltype(par)::value;
          const std::integral_constant<int, P> cur{};
          const std::integral_constant<int, 1 - P> nxt{};
          // 16 bits: V(t+1) over V(t-1), K(t+2) over K(t). 8 bits: these come out of the raw buffers in phase B, while
          // V(t+2) and K(t+3) come into the others. The rows of tile t + 1 + AHEAD are found inside phase A.
          if constexpr (k8) {
            to_raw(v_rs, rows[1], P ? v_raw1 : v_raw0);
            to_raw(k_rs, rows[2], P ? k_raw0 : k_raw1);
            scales_to_lds(t + 2, row[1]);
            l += l_next;
            l_next = 0.f;
          } else {
            to_lds(c.v, v_rs, rows[0], v_stage(nxt), true);
            to_lds(c.k, k_rs, rows[1], k_stage(cur), false);
          }
          uint64_t present_new = 0;
          int row_new = 0;
          const float inv = inverse_unit();
          // The phases are laid out by hand, one MFMA and its share of the VALU work after another (the compiler's
          // own order, and its scheduling groups, put the MFMAs first and the exponentials behind them).
          // Phase A: S(t+1) with the second half of P(t).
          __builtin_amdgcn_sched_barrier(0);
          __builtin_amdgcn_s_setprio(2);
          {
            constexpr int N = NKB * QK_STEPS, EACH = N / 4;   // MFMAs; four exponentials after each EACH of them
            const unsigned char* ks = k_stage(nxt);
            int kb = k_base;
            asm("" : "+v"(kb));
            auto operand = [&](int i) { return *reinterpret_cast<const V8*>(ks + i % NKB * 32 * RB + (kb ^ (32 * (i / NKB)))); };
            const float neg_m = neg_ref();
            V8 ahead[2] = {operand(0), operand(1)};
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const V8 x = ahead[i % 2];
              if (i + 2 < N) ahead[i % 2] = operand(i + 2);
              sn[i % NKB] = mfma32x32x16(x, qf[i / NKB], i < NKB ? f32x16{} : sn[i % NKB]);
              if (i % EACH == EACH - 1) exp_quad(s, pf, HALF * 8 + i / EACH * 4, neg_m, t, inv, l, top);
              if (i == N / 4) {
                row_new = find_row(t + 1 + AHEAD, page, in_page);
                present_new = present_of(row_new);
                page = load_page(t + 2 + AHEAD, in_page);
              }
              if (i == N / 2) {
                advance(row_new, present_new);
                chunk_rows(row_new, present_new, rows[AHEAD - 1]);
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
#pragma unroll
          for (int i = 0; i < PV_STEPS; ++i) asm volatile("" : "+v"(pf[i]));   // (not to be moved past the branch below)
          __builtin_amdgcn_s_setprio(0);
          if constexpr (kUnits) {
            // The second half outgrew its row's unit: taken again in the new one, the first half is scaled to it.
            float scaled;
            if (raise_units(top, scaled)) {
              const float neg_m = neg_ref(), inv = inverse_unit();
              float none = 0.f;
#pragma unroll
              for (int e = 0; e < HALF * 8; ++e) pf[e / 8][e % 8] = from_f32<T>(to_f32(pf[e / 8][e % 8]) * scaled);
#pragma unroll
              for (int e = HALF * 8; e < 2 * HALF * 8; e += 4) exp_quad(s, pf, e, neg_m, t, inv, none, top);
            }
            top = 0.f;
          }
          // (present[0] is tile t + 1's by now. 8 bits: masked after the scales, of which phase B then takes ones.)
          const float* ks_next = ks_lds[(t + 1) % SLOTS];
          float mx = kLowest;
          if (!is_clean(t + 1, present[0])) {
            scale_scores(sn, t + 1);
            mx = mask(sn, t + 1, present[0]);
            ks_next = ones_lds;
          }
          // Phase B: O += V(t) P(t) with the row sums of P(t), the row maxima of S(t+1) and the first half of P(t+1)
          // against the reference as it is; where that is raised after all, the half is taken again.
          {
            constexpr int N = PV_STEPS * NDB, EACH = N / 4;
            u32x4 kx[CPT], vx[CPT];
            const unsigned char* vs = v_stage(cur);
            int vb = v_base;
            asm("" : "+v"(vb));
            auto operand = [&](int i) {
              const unsigned char* p = vs + i / NDB * 16 * RB + (vb ^ (64 * (i % NDB)));
              const i16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p));
              const i16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr<i16x4>)(p + 8 * RB));
              const i16x8 x = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
              return __builtin_bit_cast(V8, x);
            };
            const float neg_m = neg_ref(), inv = inverse_unit();
            V8 ahead[2] = {operand(0), operand(1)};
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const V8 x = ahead[i % 2];
              if (i + 2 < N) ahead[i % 2] = operand(i + 2);
              o[i % NDB] = mfma32x32x16(x, pf[i / NDB], o[i % NDB]);
#pragma unroll
              for (int k = 16 * NKB / N * i; k < 16 * NKB / N * (i + 1); k += 2) {
                if constexpr (k8) {   // (four scores at a time)
                  if (k % 4 == 0) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(ks_next + k / 16 * 32 + k % 16 * 2 + 4 * hi);
#pragma unroll
                    for (int r = 0; r < 4; ++r) sn[k / 16][k % 16 + r] *= x[r];
                  }
                }
                mx = max_nan(mx, max_nan(sn[k / 16][k % 16], sn[k / 16][k % 16 + 1]));
              }
              if (i % EACH == EACH - 1) exp_quad(sn, pn, i / EACH * 4, neg_m, t + 1, inv, l_next, top);
              if constexpr (k8) {
                if (i == 0) from_raw(P ? k_raw1 : k_raw0, kx);
                if (i == N / 4) widen(kx, k_stage(cur), false);
                if (i == N / 2) from_raw(P ? v_raw0 : v_raw1, vx);
                if (i == N / 2 + N / 4) widen(vx, v_stage(nxt), true);
              } else {
#pragma unroll
                for (int k = 4 * PV_STEPS / N * i; k < 4 * PV_STEPS / N * (i + 1); ++k)
                  l = add_pair(__builtin_bit_cast(u32x4, pf[k / 4])[k % 4], l, static_cast<T*>(nullptr));
              }
              __builtin_amdgcn_sched_barrier(0);
            }
            mx = max_nan(mx, partner32(mx)) * w.scale_log2;
#pragma unroll
            for (int i = 0; i < HALF; ++i) asm volatile("" : "+v"(pn[i]));   // (not to be moved into the branches below)
          }
          settle_first(sn, pn, t + 1, raise(mx));
          __builtin_amdgcn_s_waitcnt(0);
          if (t + 1 < nt && !whole_tile(t + 1, present[0])) check_values(t + 1, v_stage(nxt));
          __syncthreads();
        };
        while (true) {
          iteration(even, t0, sa, sb, pa, pb);
          if (!fits(++t0, present[0])) break;
          iteration(odd, t0, sb, sa, pb, pa);
          if (!fits(++t0, present[0])) break;
        }
      }
    }

    find_mine();
    // ---- the tiles that the pipeline left: from the first one on that has a value that is not finite and a row that
    // does not see all of it, and all of an 8-bit WIDE cache. One by one; K(t+1) and V(t+1) arrive meanwhile, 8-bit rows
    // through registers.
#pragma unroll 1
    for (int t = t0; t < nt; ++t) {
      const int P = t & 1;
      unsigned char* const k_cur = P ? k_lds1 : k_lds0;
      unsigned char* const v_cur = P ? v_lds1 : v_lds0;
      unsigned char* const k_nxt = P ? k_lds0 : k_lds1;
      unsigned char* const v_nxt = P ? v_lds0 : v_lds1;
      const bool fetch = t + 1 < nt;
      u32x4 kx[CPT], vx[CPT];
      float scale = 0.f;
      if (fetch) {
        if constexpr (k8) {
          to_regs(c.k, k_rs, rows[0], kx);
          to_regs(c.v, v_rs, rows[0], vx);
          scale = load_scale(row[0]);
        } else {
          to_lds(c.k, k_rs, rows[0], k_nxt, false);
          to_lds(c.v, v_rs, rows[0], v_nxt, true);
        }
      }
      const uint64_t pres = present[0];
      {
        const int row_new = find_row(t + 1 + AHEAD, page, in_page);
        page = load_page(t + 2 + AHEAD, in_page);
        const uint64_t present_new = present_of(row_new);
        advance(row_new, present_new);
        chunk_rows(row_new, present_new, rows[AHEAD - 1]);
      }
      if (t < wave_tiles) {
        f32x16 s[NKB];
        V8 pf[PV_STEPS];
        const bool clean = is_clean(t, pres);
        qk(s, k_cur);
        scale_scores(s, t);
        raise(row_max(s, clean ? kLowest : mask(s, t, pres)));
        if constexpr (k8) {
          float sum, top, scaled;
          do exponentiate8(s, pf, t, sum, top); while (raise_units(top, scaled));
          l += sum;
        } else {
          exponentiate(s, pf);
        }
        if (!clean && skip_from == INT32_MAX && !values_finite(t)) skip_from = t;
        if (clean || skip_from == INT32_MAX) pv(pf, v_cur);
        if constexpr (!k8) row_sum(pf);
      }
      if constexpr (k8) {
        if (fetch) {
          widen(kx, k_nxt, false);
          widen(vx, v_nxt, true);
          store_scale(t + 1, scale);
        }
        __syncthreads();
      } else {
        __builtin_amdgcn_s_waitcnt(0);
      }
      if (fetch) check_values(t + 1, v_nxt);
      __syncthreads();
    }

    // ---- P . V of the tiles left out, over the visible pairs alone: scores again, all in fp32. Then, with fp16 rows, the
    // infinite values of a small weight: P is 0 in fp16 below 2^-25, and 0 x infinity a NaN where any positive weight makes
    // an infinity. Elements of O that are NaN in a row that is not are taken again over the values that are not finite
    // (the others make no difference to them). 4096 tokens at the end of 16384 with one such value, D = 128: 2.65 ms for
    // 1.02. Without one, a maximum over O.
    constexpr bool kInfinite = std::is_same<T, f16>::value && !k8;
    int from = skip_from;
    bool again = false;
#pragma unroll 1
    while (true) {
#pragma unroll 1
      for (int t = from; t < wave_tiles; ++t) {
        int rest;
        const int page_t = load_page(t, rest), row_t = find_row(t, page_t, rest);
        uint64_t keys = __builtin_amdgcn_ballot_w64(row_t >= 0);
        if (kInfinite && again) {
          u16x2 largest = {0, 0};
          if (row_t >= 0)
#pragma unroll 1
            for (int i = 0; i < D / 8; ++i)
              largest = max_bits(largest, *reinterpret_cast<const u32x4*>(static_cast<const C*>(c.v) + (int64_t)row_t * D + 8 * i));
          keys = __builtin_amdgcn_ballot_w64(max(largest[0], largest[1]) >= kInfBits<T>);
        } else if (is_clean(t, keys)) {
          continue;
        }
#pragma unroll 1
        for (; keys != 0; keys &= keys - 1) {
          const int k = __builtin_ctzll(keys), at = __builtin_amdgcn_readlane(row_t, k);
          const bool vis = key_begin + t * BN + k < seen;
          float dot = 0.f, x[8], ks = 1.f, vs = 1.f;
          if constexpr (k8) ks = c.k_scale[at], vs = c.v_scale[at];
#pragma unroll
          for (int kk = 0; kk < QK_STEPS; ++kk) {
            cached8(static_cast<const C*>(c.k) + (int64_t)at * D, 16 * kk + 8 * hi, 1.f, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) dot = fmaf(to_f32(qf[kk][j]), x[j], dot);
          }
          dot += partner32(dot);
          float p = exp2_fast(fmaf(dot, ks * w.scale_log2, m_run == -INFINITY ? 0.f : -m_run));
          p = vis ? p * vs : 0.f;
          if constexpr (kUnits) p *= __builtin_amdgcn_rcpf(unit);
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            cached8(static_cast<const C*>(c.v) + (int64_t)at * D, 8 * i, 1.f, x);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float y = hi ? x[4 + r] : x[r];
              if (kInfinite && again) y = fabsf(y) < INFINITY ? 0.f : y;
              o[i / 4][i % 4 * 4 + r] = fmaf(p, vis ? y : 0.f, o[i / 4][i % 4 * 4 + r]);
            }
          }
        }
      }
      if (!kInfinite || again) break;
      float any = 0.f;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; r += 2) any = max_nan(any, max_nan(o[db][r], o[db][r + 1]));
      again = __builtin_amdgcn_ballot_w64(any != any && mine && l == l) != 0;
      if (!again) break;
      from = 0;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = l == l && o[db][r] != o[db][r] ? 0.f : o[db][r];
    }

    find_mine();
    // ---- the wave's 32 rows: done, or a part for the join. (The stages are free: every wave passed the last barrier.)
    const int64_t offset = mine ? (int64_t)(sg.rows.first + token) * a.o_token + hq * a.o_head : -1;
    const bool was_mine = mine;
    const bool done = sg.from == 0 && sg.to == sg.steps;
    const int slot = sg.from == 0 ? 1 : 0;
    if (!done) {
      if (sg.from == 0) rec = {sg.seq, sg.head, sg.tile, rec.flags | kPartBegins};
      else rec.flags |= kPartContinues | (sg.to == sg.steps ? kPartEnds : 0);
    }
    {
    more = begin_segment();
    // Each wave turns its rows round in LDS of its own (a quarter or an eighth of the stages, chunks swizzled by
    // row), so that whole rows are stored, 16 bytes a lane; a lane's pieces stored as they are cost ~4 us a tile.
    int ln = (int)threadIdx.x % kWave;   // (offsets made from it are not to be hoisted out of the segments' loop)
    asm volatile("" : "+v"(ln));
    const int lq = ln % 32, hi = ln / 32, lane = ln;
    const float sum = half_sum(l);
    const float factor = done ? unit / sum : unit, nothing = m_run == -INFINITY ? 0.f : NAN;
    constexpr int PASSES = 2;   // fp32 rows: half of the wave's rows at a time
    unsigned char* const own = (wave % 4 == 0 ? k_lds0 : wave % 4 == 1 ? v_lds0 : wave % 4 == 2 ? k_lds1 : v_lds1) + wave / 4 * (32 * RB);
    if (done) {
      typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          T4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = from_f32<T>(sum == 0.f ? nothing : o[db][4 * q4 + r] * factor);
          *reinterpret_cast<T4*>(own + lq * RB + (((4 * db + q4) ^ lq % CR) * 16) + 8 * hi) = x;
        }
#pragma unroll
      for (int i = 0; i < 32 * CR / kWave; ++i) {
        const int r = (i * kWave + lane) / CR, ch = (i * kWave + lane) % CR;
        const u32x4 x = *reinterpret_cast<const u32x4*>(own + r * RB + ((ch ^ r % CR) * 16));
        const int64_t at = (int64_t)(unsigned)__shfl((int)offset, r) | (int64_t)__shfl((int)(offset >> 32), r) << 32;
        if (at >= 0) *reinterpret_cast<u32x4*>(static_cast<T*>(a.o) + at + 8 * ch) = x;
      }
    } else {
      const uint64_t rows_here = __builtin_amdgcn_ballot_w64(was_mine);
      float* const to = part_rows(w, wg, slot, BM, D) + 32 * wave * D;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        if (lq / 16 == p)
#pragma unroll
          for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              f32x4 x;
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = o[db][4 * q4 + e] * factor;
              *reinterpret_cast<f32x4*>(own + lq % 16 * (2 * RB) + (((8 * db + 2 * q4 + hi) ^ lq % 16) * 16)) = x;
            }
#pragma unroll
        for (int i = 0; i < 16 * 2 * CR / kWave; ++i) {
          const int r = (i * kWave + lane) / (2 * CR), ch = (i * kWave + lane) % (2 * CR);
          const f32x4 x = *reinterpret_cast<const f32x4*>(own + r * (2 * RB) + ((ch ^ r) * 16));
          if (rows_here >> (16 * p + r) & 1) *reinterpret_cast<f32x4*>(to + (16 * p + r) * D + 4 * ch) = x;
        }
      }
      if (was_mine && hi == 0) {
        const int r = 32 * wave + lq;
        float* st = part_stats(w, (int)gridDim.x, wg, slot, BM, D);
        // (Scores that are all NaN leave no maximum and a NaN sum, which must not count as a row that sees nothing.)
        st[r] = m_run == -INFINITY && sum != 0.f ? 0.f : m_run, st[BM + r] = sum;
      }
    }
    }
    __syncthreads();   // the next segment's loads replace the stages
  }
  if (tid == 0) w.records[wg] = rec;
}

// Joins the parts of the tile that workgroup blockIdx.x of the attention kernel began and did not end: its own
// and those of the workgroups after it, up to the one that ends the tile. 16 threads a row. What bounds it is
// the latency of its loads, so that no load waits for another but the records: the parts' number comes from
// 64 records at once, their weights by lane, and their rows four parts at a time. 4.5 to 6.3 us after tiles of few rows
// (kernels of 10 to 220 us); after chunks, whose parts are 45 to 67 MB, 14 to 17 (kernels of 74 to 2090).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(256) paged_attn_join(PagedCache c, RowsQ a, AttnWork w, int wgs) {
  constexpr int EL = D / 16, MOST = 64;
  __shared__ float weight[16][MOST];
  const int first = (int)blockIdx.x, lane = (int)threadIdx.x % kWave;
  const PartRecord rec = w.records[first];
  if (!(rec.flags & kPartBegins)) return;
  int n = 1;   // parts
  for (int at = first + 1; at < wgs; at += kWave) {
    const int flags = at + lane < wgs ? w.records[at + lane].flags : kPartEnds;
    const uint64_t ends = __builtin_amdgcn_ballot_w64((flags & kPartEnds) != 0);
    n = at - first + (ends ? __builtin_ctzll(ends) + 1 : kWave);
    if (ends) break;
  }
  n = min(n, wgs - first);
  const SeqRows s = load_seq(c, rec.seq);
  const int part = (int)threadIdx.x % 16, tr = (int)threadIdx.x / 16;
  for (int r0 = (int)blockIdx.y * 16; r0 < ROWS; r0 += (int)gridDim.y * 16) {
    const int r = r0 + tr;
    int token, hq;
    const bool mine = tile_row(w.tiles, s, rec.head, rec.tile, in_tile(w.tiles, r), token, hq);
    float m = -INFINITY, sum = 0.f, x[EL] = {};
    for (int p0 = 0; p0 < n; p0 += MOST) {
      float mi[MOST / 16], li[MOST / 16], top = -INFINITY, add = 0.f;
#pragma unroll
      for (int k = 0; k < MOST / 16; ++k) {
        const int i = p0 + 16 * k + part;
        mi[k] = -INFINITY, li[k] = 0.f;
        if (mine && i < n) {
          const float* st = part_stats(w, wgs, first + i, i == 0 ? 1 : 0, ROWS, D);
          mi[k] = st[r], li[k] = st[ROWS + r];
        }
      }
#pragma unroll
      for (int k = 0; k < MOST / 16; ++k) top = fmaxf(top, mi[k]);
      top = fmaxf(top, dpp_move<0xB1>(top));
      top = fmaxf(top, dpp_move<0x4E>(top));
      top = fmaxf(top, dpp_move<0x141>(top));
      top = fmaxf(top, dpp_move<0x140>(top));
      const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.f : exp2_fast(m - mn);
#pragma unroll
      for (int k = 0; k < MOST / 16; ++k) {
        const float e = mi[k] == -INFINITY ? 0.f : exp2_fast(mi[k] - mn);
        weight[tr][16 * k + part] = e;
        add = fmaf(e, li[k], add);
      }
      add += dpp_move<0xB1>(add);
      add += dpp_move<0x4E>(add);
      add += dpp_move<0x141>(add);
      add += dpp_move<0x140>(add);
      sum = sum * f + add;
      m = mn;
#pragma unroll
      for (int e = 0; e < EL; ++e) x[e] = f > 0.f ? x[e] * f : 0.f;
      // (A row's weights are written and read by the same wave, in order.)
      if (mine)
#pragma unroll 4
        for (int i = 0; i < min(MOST, n - p0); ++i) {
          const float wi = weight[tr][i];
          const float* from = part_rows(w, first + p0 + i, p0 + i == 0 ? 1 : 0, ROWS, D) + r * D + part * EL;
#pragma unroll
          for (int e = 0; e < EL; e += 4) {
            const f32x4 y = *reinterpret_cast<const f32x4*>(from + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[e + j] = fmaf(wi, wi > 0.f ? y[j] : 0.f, x[e + j]);
          }
        }
    }
    if (!mine) continue;
    typedef T TE __attribute__((ext_vector_type(EL)));
    TE y;
#pragma unroll
    for (int e = 0; e < EL; ++e) y[e] = from_f32<T>(row_result(x[e], m, sum));
    *reinterpret_cast<TE*>(static_cast<T*>(a.o) + (int64_t)(s.first + token) * a.o_token + hq * a.o_head + part * EL) = y;
  }
}

}  // namespace pa
