// Attention of packed query rows over the 8-bit paged K/V cache (kv_cache.hip
// has its layout): decode, verify and prompt chunks of grouped-query heads,
// causal, with an optional sliding window.
//
//   s_j = scale * ks(page j) * (q . kcode_j),   p_j = exp(s_j - m) over the
//   visible j, out = sum_j p_j vs(page j) vcode_j / sum_j p_j
//
// One pass over the cache with the running maximum and sum of a softmax.  The
// G query heads of a kv head and the rows of a request are the columns of one
// product: tile column r is row r / G, head r % G, so K and V are read once for
// all of them.
//
// Bound by memory where rows are few, and there by how evenly the items keep the chip
// reading: 1024 requests of 2000 tokens, 16 + 8 heads of 256, read 5.7 TB/s (the call, 1484
// us), 47 of 33 to 8190 tokens 4.9 (161 us), two of 70001 and 130005 tokens, 16 + 2 heads of
// 512, 5.1 (80 us); a plain read reaches 6.6 to 6.8 over as many bytes.  Bound by issue
// where rows are many (2048 rows on 8100 tokens: 263 to 312 us by box, 900 to 760 TFLOP/s;
// matrix cores busy 37%, one wave a SIMD), by the start and end of a round of workgroups
// between (9 requests of 7 rows on 600 to 5000 tokens of width 512: 34 us, of
// which 17 without a unit).

#include "../../include/gemmainfer_amd.h"
#include "gi_common.h"
#include "gi_internal.h"

namespace gi {

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kUnit = 64;      // cache rows a wave takes at a time
constexpr int kMinChunk = 4;   // units: one a wave
constexpr int kRounds = 4;
constexpr int kEnds = 64;      // bytes of the plan in front of the running counts
// what a compute unit holds of a kernel: by its registers, two waves a SIMD or one
constexpr int workgroups_per_cu(int D, int CT) { return D * CT <= (CT == 1 ? 256 : 128) ? 2 : 1; }
constexpr float kLog2e = 1.4426950408889634f;
// The partial sums fit the workspace while choose_chunk's total is right to 1e-4: over this
// many requests, 1024 to a thread, an fp32 sum is off by at most about 2^10 * 2^-24.
constexpr int kMaxRequests = 1 << 20;
constexpr int kMaxGrid = 1 << 23;  // workgroups: with their threads under the 2^32 that a launch may have
// Weights go to the matrix cores in fp16 as 2^(t - m + kBias).  The reference m
// is a maximum of earlier rows and follows when a lane's 16 weights sum to more than
// kMostSum, so none is over fp16's largest; fp16 is normal down to 2^-14, so a weight
// 2^-25 of that of m still has all 11 bits, and a lighter one is off by at most 2^-36 of
// it: a flat tail behind one heavy token loses less than half a step of fp16 (2^-11)
// over 2^25 tokens.  With a bias of 3 (2^-28) the sums could grow 2^8 times as much
// before the reference follows: 2048 rows on 8100 tokens 272 instead of 285 us where
// scores are spread widely (deviation 6), 274 instead of 266 where they are not (1.5).
constexpr float kBias = 11.f;
constexpr float kMostSum = 65504.f;

struct AttnArgs {
  const void* q;
  int64_t q_st, q_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  const float* ks;
  const float* vs;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* q_start;  // null: one row a request
  void* out;
  int64_t o_st, o_sh;
  int* plan;               // the chunk; at kEnds bytes, for more than 64 requests, int4 [B] running counts
  float* part;             // [max_slots * Hk][RT][D] partial sums, then [max_slots * Hk][RT] (maximum, sum)
  int64_t num_pages;
  float scale;             // with log2(e)
  int T, B, Hk, G, cols, log_page, window;
  int resident;            // workgroups of a kv head that the chip holds at a time
  int max_slots;
};

// ---------------------------------------------------------------------------
// the work list
// ---------------------------------------------------------------------------
// An item is (request, tile of RT columns, chunk of units); every workgroup
// finds its own from the request lengths, on the device, so the launch needs no
// host copy of them and can be replayed from a graph for other lengths.  The
// chunk is the same for all requests: a long one is shared by as many
// workgroups as a batch of short ones.  Up to 64 requests are one load of a
// wave; for more, a workgroup launched first writes the chunk and running counts of
// items, tiles and partial sums, and the others search those.
struct Item {
  int b, tile, chunk_no, chunk, q0, rows, len;
  int slot;   // of the tile's first partial sum, among those of one kv head
  bool over;  // longer than the table: its pages cannot all be there
};

// The lane, worked out anew: what hangs on it in the loop over items is not
// kept in registers from one to the next.
__device__ __forceinline__ int this_lane() {
  int v = threadIdx.x & 63;
  asm volatile("" : "+v"(v));
  return v;
}

struct Load {  // of one request
  int q0, rows, len, tiles, units;
  bool over;
};

template <int RT>
__device__ __forceinline__ Load load_of(const AttnArgs& a, int b) {
  Load r{0, 0, 0, 0, 0, false};
  if (b >= a.B) return r;
  int q0 = b, q1 = b + 1;
  if (a.q_start) {
    q0 = min(max(a.q_start[b], 0), a.T);
    q1 = min(max(a.q_start[b + 1], q0), a.T);
  }
  const int cap = a.cols << a.log_page;  // at most 2^30
  const int len = max(a.lens[b], 0);
  r.q0 = q0;
  r.rows = q1 - q0;
  r.over = len > cap;
  r.len = min(len, cap);
  r.tiles = (r.rows * a.G + RT - 1) / RT;  // rows * G at most 2^30
  r.units = (r.len + kUnit - 1) / kUnit;
  if (a.window > 0) r.units = min(r.units, (a.window + RT) / kUnit + 2);  // a window is shorter than the table
  return r;
}

__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// ceil(n / d), n + d at most 2^25: a quotient in fp32 is off by one at most.
__device__ __forceinline__ int ceil_div(int n, int d) {
  n += d - 1;
  int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
  const int r = n - q * d;
  q += r >= d ? 1 : 0;
  return r < 0 ? q - 1 : q;
}

// The chunk, in units: the tile units of a kv head go to `resident` workgroups
// that the chip holds at a time, in k = 1 ... 4 rounds.  One round
// is best where the chunks come out even (a few long requests: two of 70001 and 130005
// tokens 93 us with the join in one round, 112 in two), several where many requests of
// other lengths leave workgroups idle (47 up to 8190 tokens: 186, 173, 173 and 175 us in
// one to four).  k is the one with the least estimate: rounds of whole
// chunks, or what any order of work stays under, and two units to start each round.
// `sum` adds a number of each request up.
template <typename Sum>
__device__ __forceinline__ int choose_chunk(const AttnArgs& a, Sum&& sum) {
  const float total = sum([](const Load& l) { return (float)l.tiles * (float)l.units; });
  // not less than the exact total, whatever was rounded: chunk >= total / (k * resident)
  const float each = total * 1.0001f * __builtin_amdgcn_rcpf((float)a.resident);
  int best = 0;
  float least = 0.f;
#pragma unroll 1
  for (int k = 1; k <= kRounds; ++k) {
    // a chunk of 2^24 units holds any request
    int c = (int)fminf(each * __builtin_amdgcn_rcpf((float)k), 16777200.f) + 1;
    c = (max(c, kMinChunk) + kWaves - 1) / kWaves * kWaves;
    if (k > 1 && c >= best) break;
    const float items = sum([c](const Load& l) { return (float)l.tiles * (float)ceil_div(l.units, c); });
    const float rounds = ceilf(items * __builtin_amdgcn_rcpf((float)a.resident));
    const float cost = fminf(rounds * c, each + c) + 2.f * rounds;
    if (k == 1 || cost < least) {
      best = c;
      least = cost;
    }
    if (c <= 4 * kMinChunk) break;
  }
  return __builtin_amdgcn_readfirstlane(best);
}

struct Counts {
  int items, tiles, slots;
};

__device__ __forceinline__ Counts counts_of(const Load& l, int chunk) {
  const int chunks = max(ceil_div(l.units, chunk), 1), n = l.tiles * chunks;
  return Counts{n, l.tiles, chunks > 1 ? n : 0};
}

// The chunk of up to 64 requests: every workgroup finds the same.
template <int RT>
__device__ __forceinline__ int chunk_of_few(const AttnArgs& a) {
  const Load mine = load_of<RT>(a, threadIdx.x & 63);
  return choose_chunk(a, [&](auto&& number) { return wave_sum_f32(number(mine)); });
}

// The plan of more: one workgroup.
constexpr int kPlanThreads = 1024;
template <int RT>
__global__ __launch_bounds__(kPlanThreads) void kv_attention_plan_kernel(AttnArgs a) {
  __shared__ float part[kPlanThreads / kWave];
  __shared__ int sums[3][kPlanThreads / kWave];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int chunk = choose_chunk(a, [&](auto&& number) {
    float v = 0.f;
    for (int b = tid; b < a.B; b += kPlanThreads) v += number(load_of<RT>(a, b));
    v = wave_sum_f32(v);
    __syncthreads();  // the sum before is read
    if ((tid & 63) == 0) part[wave] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < kPlanThreads / kWave; ++w) v += part[w];
    return v;
  });
  if (tid == 0) *a.plan = chunk;
  int4* ends = (int4*)((char*)a.plan + kEnds);
  int carry[3] = {0, 0, 0};
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const Counts c = counts_of(load_of<RT>(a, b0 + tid), chunk);
    int v[3] = {wave_scan(c.items), wave_scan(c.tiles), wave_scan(c.slots)};
    __syncthreads();
    if ((tid & 63) == 63)
      for (int x = 0; x < 3; ++x) sums[x][wave] = v[x];
    __syncthreads();
    for (int x = 0; x < 3; ++x) {
      int all = 0;
      for (int w = 0; w < kPlanThreads / kWave; ++w) {
        if (w == wave) v[x] += carry[x] + all;
        all += sums[x][w];
      }
      carry[x] += all;
    }
    if (b0 + tid < a.B) ends[b0 + tid] = make_int4(v[0], v[1], v[2], 0);
  }
}

// Item `want` of the list (by_tile: the first item of tile `want`); false past its end.
template <int RT>
__device__ __forceinline__ bool find_item(const AttnArgs& a, int chunk, int want, bool by_tile, Item& it) {
  const int lane = this_lane();
  int in, slot;
  Load l;
  if (a.B <= kWave) {
    const Load mine = load_of<RT>(a, lane);
    const Counts c = counts_of(mine, chunk);
    const int count = by_tile ? c.tiles : c.items;
    const int end = wave_scan(count), slot_end = wave_scan(c.slots);
    const unsigned long long hit = __ballot(want >= end - count && want < end);
    if (!hit) return false;
    it.b = __ffsll(hit) - 1;
    auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, it.b); };
    in = want - pick(end - count);
    slot = pick(slot_end - c.slots);
    l = Load{pick(mine.q0), pick(mine.rows), pick(mine.len), pick(mine.tiles), pick(mine.units), pick((int)mine.over) != 0};
  } else {
    // the first request whose running count is over `want`: 64 of them at a time, then those up to it
    const int4* ends = (const int4*)((const char*)a.plan + kEnds);
    auto end_of = [&](int b) { return by_tile ? ends[b].y : ends[b].x; };
    const int step = (a.B + kWave - 1) / kWave;
    unsigned long long over = __ballot(end_of(min((lane + 1) * step, a.B) - 1) > want);
    if (!over) return false;
    const int lo = (__ffsll(over) - 1) * step, hi = min(lo + step, a.B);
    for (int b0 = lo;; b0 += kWave) {
      over = __ballot(end_of(min(b0 + lane, hi - 1)) > want);
      it.b = min(b0 + (over ? __ffsll(over) - 1 : 0), hi - 1);
      if (over || b0 + kWave >= hi) break;
    }
    const int4 before = it.b > 0 ? ends[it.b - 1] : make_int4(0, 0, 0, 0);
    in = want - (by_tile ? before.y : before.x);
    slot = before.z;
    l = load_of<RT>(a, it.b);
    // requests that share rows (offsets that decrease) can be more than the counts hold
    if (in < 0 || in >= l.tiles * (by_tile ? 1 : max(ceil_div(l.units, chunk), 1))) return false;
  }
  const int per = max(ceil_div(l.units, chunk), 1);
  const int tile = by_tile ? in : in / per;
  it.chunk_no = by_tile ? 0 : in - tile * per;
  it.chunk = chunk;
  it.q0 = l.q0;
  it.rows = l.rows;
  it.len = l.len;
  it.over = l.over;
  it.slot = slot + tile * per;
  it.tile = l.tiles - 1 - tile;  // the last tiles of a prompt see the most: they go first
  for (int* f : {&it.b, &it.tile, &it.chunk_no, &it.q0, &it.rows, &it.len, &it.slot})
    *f = __builtin_amdgcn_readfirstlane(*f);
  return true;
}

// What a tile's columns see: units [lo, hi), and how many chunks they are cut into.
struct Span {
  int lo, hi, chunks;
  int pos_min, pos_max;  // positions of its first and last row
};

template <int RT>
__device__ __forceinline__ Span span_of(const AttnArgs& a, const Item& it) {
  Span s;
  const int r0 = it.tile * RT, r1 = min(r0 + RT, it.rows * a.G) - 1;
  s.pos_min = it.len - it.rows + r0 / a.G;
  s.pos_max = it.len - it.rows + r1 / a.G;
  s.lo = 0;
  if (a.window > 0) s.lo = max(s.pos_min - a.window + 1, 0) / kUnit;
  s.hi = s.pos_max < 0 ? 0 : s.pos_max / kUnit + 1;
  s.chunks = max(ceil_div(s.hi - s.lo, it.chunk), 1);
  return s;
}

// ---------------------------------------------------------------------------
// types of the first product (the second one is fp16 for both)
// ---------------------------------------------------------------------------
template <bool F16>
struct Qk;
template <>
struct Qk<false> {
  typedef bf16x8_t frag;
  static __device__ __forceinline__ frag codes(uint32_t lo, uint32_t hi) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
    return frag{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  static __device__ __forceinline__ f32x4_t mfma(frag a, frag b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t out(float f) { return f32_to_bf16(f); }
};

__device__ __forceinline__ f16x8_t codes_f16(uint32_t lo, uint32_t hi) {
  const f16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
  const f16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
  const f16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
  const f16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  return f16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f32x4_t mfma_f16(f16x8_t a, f16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <>
struct Qk<true> {
  typedef f16x8_t frag;
  static __device__ __forceinline__ frag codes(uint32_t lo, uint32_t hi) { return codes_f16(lo, hi); }
  static __device__ __forceinline__ f32x4_t mfma(frag a, frag b, f32x4_t c) { return mfma_f16(a, b, c); }
  static __device__ __forceinline__ uint16_t out(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }
};

// ---------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// max over the four lanes of a column (lane % 16), to all of them
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// What a wave reads of one unit.
struct UnitRef {
  const uint8_t* k;
  const uint8_t* v;
  float ks, vs;
};

// The four waves of a workgroup take turns at units of 64 cache rows; each has
// its own running softmax over 16 * CT columns, joined at the end through LDS.
// No barrier in the loop, and K and V do not pass through LDS: lane (i = lane %
// 16, g = lane / 16) reads from the cache just what its place in the MFMA
// operands needs.
//   S^T = K Q^T, 16x16x32: operand A's row i of product j is cache row 16 (i / 4) +
//     4 j + i % 4 of the unit, so that the four results of lane (i, g) are rows
//     16 g + 4 j ... + 3 of column i: after j = 0..3 a lane holds the 16
//     rows of ITS group g, one page's rows, in order.
//   O^T = V^T P^T: operand B wants 8 rows of column i from lane (i, g): those
//     are its own scores.  Operand A is 16 rows of dimension 16 dt + i, one
//     16-byte load of the transposed V.
// So neither the scores nor V cross lanes, and a lane needs one K and one V
// scale per unit.  A column's maximum is the only exchange (two lane swaps).
//
// A unit is D / 64 steps of K and as many of V, each 64 dimensions of 64 rows in four loads a
// lane.  The loads of the next kRing - 1 steps are always in flight, over the
// end of a unit as well, so the matrix cores and the softmax run while HBM (or
// L2) delivers.  A K step meets its two Q operands of a column tile with all
// four products, so Q from LDS (where it does not fit in registers) is read once a unit.
//
// V's scale joins the exponent: t = s + log2(vs), weights 2^(t - m), m over t.
// The sum of softmax weights is then sum 2^(t - m) / vs.  With it the weights
// of V's codes stay in fp16's range whatever the scales are, and the
// maximum is over what each row can contribute.  Most units need no maximum at
// all: their weights are formed with the reference there is, and only where a sum
// shows that one has grown too large are the maximum found, the sums scaled and the weights
// formed again.
template <int D, int CT, bool F16>
__global__ __launch_bounds__(kThreads, workgroups_per_cu(D, CT)) void kv_attention_kernel(AttnArgs a) {
  constexpr int RT = 16 * CT;
  constexpr int KS = D / 64;   // steps of K, and of V: 64 dimensions, four 16-byte loads of a lane
  constexpr int DT = D / 16;   // dimension tiles of the output
  constexpr int kSteps = 2 * KS;
  constexpr int kRing = D == 64 ? 2 : D == 512 ? 8 : 4;
  constexpr bool kQLds = CT * D > 512;
  // the waves' sums meet in LDS, a part of the dimensions at a time where they do not fit together
  constexpr int kParts = (size_t)RT * (D + 4) * kWaves * 4 <= 140000 ? 1 : 2;
  constexpr int DP = D / kParts, kPitch = DP + 4;
  // What may move over a step's loads: nothing, or where a compute unit holds
  // two workgroups all that is no memory access (16 columns of 256: 173 us instead of
  // 176; where it holds one, the other way: 64 columns of 256 268 instead of 357, 32 of
  // 512 41 instead of 67)
  constexpr int kFree = workgroups_per_cu(D, CT) > 1 ? 0x8f : 0;
  constexpr size_t kRedBytes = (size_t)kWaves * RT * kPitch * 4, kQBytes = kQLds ? (size_t)CT * 2 * KS * kWave * 16 : 16;
  typedef typename Qk<F16>::frag frag;
  __shared__ __align__(16) char lds[kRedBytes > kQBytes ? kRedBytes : kQBytes];
  __shared__ float red_m[kWaves][RT], red_l[kWaves][RT];
  uint4* q_lds = (uint4*)lds;
  float* red = (float*)lds;

  const int wave = uniform(threadIdx.x >> 6);
  const int hk = blockIdx.x % a.Hk;
  const int chunk = a.B <= kWave ? chunk_of_few<RT>(a) : *a.plan;
  if (a.B <= kWave && blockIdx.x == 0 && threadIdx.x == 0) *a.plan = chunk;  // for the join
  Item it;
  for (int want = blockIdx.x / a.Hk; find_item<RT>(a, chunk, want, false, it); want += gridDim.x / a.Hk) {
  const Span sp = span_of<RT>(a, it);
  const int r0 = it.tile * RT, n_cols = min(RT, it.rows * a.G - r0);
  // longer than the table, or (which choose_chunk's total rules out) without room for its partial sums
  const bool lost = it.over || (sp.chunks > 1 && it.slot + sp.chunks > a.max_slots);
  if (lost) {
    if (it.chunk_no == 0) {
      const uint32_t nan = F16 ? 0x7e007e00u : 0x7fc07fc0u;
      for (int e = threadIdx.x; e < n_cols * (D / 8); e += kThreads) {
        const int c = e / (D / 8), r = r0 + c, row = r / a.G, head = hk * a.G + (r - row * a.G);
        *(uint4*)((uint16_t*)a.out + (it.q0 + row) * a.o_st + head * a.o_sh + (e - c * (D / 8)) * 8) =
            make_uint4(nan, nan, nan, nan);
      }
    }
    continue;
  }
  if (it.chunk_no >= sp.chunks) continue;
  __syncthreads();  // the item before is done with LDS
  const int lane = this_lane();
  const int i16 = lane & 15, g = lane >> 4;
  const int page_mask = (1 << a.log_page) - 1;

  // ---- Q as operand B: column i, dimensions 64 s + 16 g + 8 h ... of step 2 s + h
  frag qf[kQLds ? 1 : CT][kQLds ? 1 : 2 * KS];
  int hi_pos[CT];  // the column's position: it sees rows up to it
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = ct * 16 + i16, r = r0 + min(c, n_cols - 1);
    const int row = r / a.G, head = hk * a.G + (r - row * a.G);
    hi_pos[ct] = it.len - it.rows + row;
    const uint16_t* src = (const uint16_t*)a.q + (it.q0 + row) * a.q_st + head * a.q_sh;
#pragma unroll
    for (int s = 0; s < 2 * KS; ++s) {
      if (kQLds && (ct * 2 * KS + s) % kWaves != wave) continue;
      const uint4 w = *(const uint4*)(src + (s >> 1) * 64 + g * 16 + (s & 1) * 8);
      if (kQLds) q_lds[(s * CT + ct) * kWave + lane] = w;
      else qf[kQLds ? 0 : ct][kQLds ? 0 : s] = __builtin_bit_cast(frag, w);
    }
  }
  if (kQLds) __syncthreads();

  f32x4_t acc[CT][DT];
  float m[CT], l[CT];  // the reference of the weights (-inf: none yet), their sum over v's scale
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[ct][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* table = a.table + it.b * a.table_stride;
  const int grp_k = 16 * (i16 >> 2);
  auto page_of = [&](int tok) -> int {
    const int col = tok >> a.log_page;
    return col < a.cols ? table[col] : -1;
  };
  auto ref_of = [&](int u, int kp, int vp) -> UnitRef {
    const int tok = u * kUnit;
    // a page that is not there: nothing is read from where it points, and its
    // rows, if they are seen at all, have no scale
    const int64_t kq = kp < 0 || kp >= a.num_pages ? 0 : kp;
    const bool bad = vp < 0 || vp >= a.num_pages;
    const int64_t vq = bad ? 0 : vp;
    UnitRef r;
    r.k = a.kc + (((kq * a.Hk + hk) << a.log_page) + ((tok + grp_k) & page_mask) + (i16 & 3)) * D + 16 * g;
    r.v = a.vc + (((vq * a.Hk + hk) * D + i16) << a.log_page) + ((tok + 16 * g) & page_mask);
    r.ks = a.ks[vq * a.Hk + hk];
    r.vs = a.vs[vq * a.Hk + hk];
    if (bad) r.ks = r.vs = __uint_as_float(0x7fc00000u);
    return r;
  };
  const int u_end = uniform(min(sp.lo + (it.chunk_no + 1) * it.chunk, sp.hi));
  const int u_first = uniform(sp.lo + it.chunk_no * it.chunk + wave);
  const int pos_min = uniform(sp.pos_min), pos_max = uniform(sp.pos_max);

  if (u_first < u_end) {
    const int u_last = u_first + (u_end - 1 - u_first) / kWaves * kWaves;
    uint4 ring[kRing][4];
    // loads step `st` of a unit into its place of the ring
    auto issue = [&](const UnitRef& r, int st) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        ring[st % kRing][i] = st < KS ? *(const uint4*)(r.k + i * 4 * D + st * 64)
                                      : *(const uint4*)(r.v + ((size_t)(((st - KS) * 4 + i) * 16) << a.log_page));
    };
    UnitRef cur = ref_of(u_first, page_of(u_first * kUnit + grp_k), page_of(u_first * kUnit + 16 * g));
    const int u1 = min(u_first + kWaves, u_last);
    UnitRef nxt = ref_of(u1, page_of(u1 * kUnit + grp_k), page_of(u1 * kUnit + 16 * g));
#pragma unroll
    for (int st = 0; st < kRing - 1; ++st) issue(cur, st);

    for (int u = u_first; u < u_end; u += kWaves) {
      const int tok = u * kUnit;
      // past the last unit the loads repeat it (they are not used)
      const int u2 = min(u + 2 * kWaves, u_last);
      const int kp2 = page_of(u2 * kUnit + grp_k), vp2 = page_of(u2 * kUnit + 16 * g);
      const bool edge = tok + kUnit - 1 > pos_min || (a.window > 0 && tok <= pos_max - a.window);
      f32x4_t s[CT][4];
      f16x8_t p[CT][2];
      auto ahead = [&](int st) {
        if (st + kRing - 1 < kSteps) issue(cur, st + kRing - 1);
        else issue(nxt, st + kRing - 1 - kSteps);
        __builtin_amdgcn_sched_barrier(kFree);
      };

      // ---- scores
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[ct][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      uint4 q_next[3];
      if (kQLds) {
        q_next[0] = q_lds[lane];
        q_next[1] = q_lds[kWave + lane];
      }
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        ahead(st);
        frag k[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 w = ring[st % kRing][j];
          k[j][0] = Qk<F16>::codes(w.x, w.y);
          k[j][1] = Qk<F16>::codes(w.z, w.w);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            if (kQLds) {  // two operands ahead of the products: LDS takes as long as eight of them
              const int n = (2 * st + h) * CT + ct;
              if (n + 2 < 2 * KS * CT) q_next[(n + 2) % 3] = q_lds[(n + 2) * kWave + lane];
              __builtin_amdgcn_sched_barrier(0x16);
            }
            const frag q = kQLds ? __builtin_bit_cast(frag, q_next[((2 * st + h) * CT + ct) % 3])
                                 : qf[kQLds ? 0 : ct][kQLds ? 0 : 2 * st + h];
#pragma unroll
            for (int j = 0; j < 4; ++j) s[ct][j] = Qk<F16>::mfma(k[j][h], q, s[ct][j]);
          }
      }

      // ---- weights
      float c1 = cur.ks * a.scale, c0 = __log2f(cur.vs);
      const float inv_vs = 1.f / cur.vs;
      if (edge) {
        // what is not seen scores -inf, whatever its page's scale is
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int hi = hi_pos[ct] - (tok + 16 * g), lo = a.window > 0 ? hi - a.window : -1;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[ct][j][r] = 4 * j + r <= hi && 4 * j + r > lo ? fmaf(s[ct][j][r], c1, c0) : -INFINITY;
        }
        c1 = 1.f;
        c0 = 0.f;
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        auto weigh = [&]() {
          const float shift = c0 + (kBias - (m[ct] == -INFINITY ? 0.f : m[ct]));
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float w = exp2_fast(fmaf(s[ct][j][r], c1, shift));
              sum += w;
              p[ct][j >> 1][(j & 1) * 4 + r] = (_Float16)w;
            }
          return sum;
        };
        float sum = weigh();
        // the reference has to follow: a weight is near what fp16 holds, or there is none yet
        if (__any(!(sum <= kMostSum) || m[ct] == -INFINITY)) {
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, fmaf(s[ct][j][r], c1, c0));
          top = fmaxf(m[ct], column_max(top));
          if (m[ct] != -INFINITY) {
            const float f = exp2_fast(m[ct] - top);
            l[ct] *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[ct][dt] *= f;
          }
          m[ct] = top;
          sum = weigh();
        }
        // rows that are not seen weigh nothing, whatever their page's scale is
        l[ct] += sum == 0.f ? 0.f : sum * inv_vs;
      }

      // ---- O^T += V^T P^T
      // (masked in every unit: one straight line of code is scheduled better than two, 3% of the
      // instructions of 64 columns)
      // a page that is not there, or has no scale: its rows weigh NaN where they are seen and nothing where
      // they are not, and what was read in its place may hold anything
      const uint32_t all = cur.vs == cur.vs ? ~0u : 0u;
      uint32_t keep[4] = {all, all, all, all};
      if (edge) {  // rows that no column sees may hold anything
        const int last = min(pos_max - (tok + 16 * g), 15);
        const int first = a.window > 0 ? pos_min - a.window + 1 - (tok + 16 * g) : 0;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          keep[x] = 0;
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (4 * x + y <= last && 4 * x + y >= first) keep[x] |= all & 0xffu << (8 * y);
        }
      }
#pragma unroll
      for (int st = KS; st < kSteps; ++st) {
        ahead(st);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 w = ring[st % kRing][i];
          w = make_uint4(w.x & keep[0], w.y & keep[1], w.z & keep[2], w.w & keep[3]);
          const f16x8_t v0 = codes_f16(w.x, w.y), v1 = codes_f16(w.z, w.w);
          const int dt = (st - KS) * 4 + i;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[ct][dt] = mfma_f16(v0, p[ct][0], acc[ct][dt]);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[ct][dt] = mfma_f16(v1, p[ct][1], acc[ct][dt]);
        }
      }
      cur = nxt;
      nxt = ref_of(u2, kp2, vp2);
    }
  }

  // ---- join the waves
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, kWave);
    l[ct] += __shfl_xor(l[ct], 32, kWave);
    if (g == 0) {
      red_m[wave][ct * 16 + i16] = m[ct];
      red_l[wave][ct * 16 + i16] = l[ct];
    }
  }
  __syncthreads();
  float f[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red_m[w][ct * 16 + i16]);
    f[ct] = m[ct] == -INFINITY ? 0.f : exp2_fast(m[ct] - top);
    if (m[ct] == -INFINITY && l[ct] != l[ct]) f[ct] = l[ct];  // only scores without a value: they stay NaN
  }
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    if (part > 0) __syncthreads();
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int dt = 0; dt < DT / kParts; ++dt)
        *(f32x4_t*)(red + (wave * RT + ct * 16 + i16) * kPitch + dt * 16 + 4 * g) = acc[ct][part * (DT / kParts) + dt] * f[ct];
    __syncthreads();
    for (int e = threadIdx.x; e < n_cols * (DP / 8); e += kThreads) {
      const int c = e / (DP / 8), dl = (e - c * (DP / 8)) * 8, d = part * DP + dl;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, red_m[w][c]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (red_m[w][c] != -INFINITY) sum += red_l[w][c] * exp2_fast(red_m[w][c] - top);
      f32x4_t o0 = {0.f, 0.f, 0.f, 0.f}, o1 = o0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        o0 += *(const f32x4_t*)(red + (w * RT + c) * kPitch + dl);
        o1 += *(const f32x4_t*)(red + (w * RT + c) * kPitch + dl + 4);
      }
      if (sp.chunks == 1) {
        const int r = r0 + c, row = r / a.G, head = hk * a.G + (r - row * a.G);
        uint16_t o[8];
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          o[x] = Qk<F16>::out(o0[x] * inv);
          o[4 + x] = Qk<F16>::out(o1[x] * inv);
        }
        *(uint4*)((uint16_t*)a.out + (it.q0 + row) * a.o_st + head * a.o_sh + d) =
            make_uint4(o[0] | o[1] << 16, o[2] | o[3] << 16, o[4] | o[5] << 16, o[6] | o[7] << 16);
      } else {
        const size_t at = ((size_t)(it.slot + it.chunk_no) * a.Hk + hk) * RT + c;
        float* dst = a.part + at * D + d;
        *(f32x4_t*)dst = o0;
        *(f32x4_t*)(dst + 4) = o1;
        if (d == 0) {
          float* ml = a.part + (size_t)a.max_slots * a.Hk * RT * D + at * 2;
          ml[0] = top;
          ml[1] = sum;
        }
      }
    }
  }
  }
}

// Joins the chunks of tiles that were cut: out = sum_c 2^(m_c - m) O_c / sum_c
// 2^(m_c - m) l_c.  A workgroup takes 256 values at a time (64 lanes of four
// dimensions); its waves take a quarter of the chunks each, and their sums meet
// in LDS, in order.
template <int D, int CT, bool F16>
__global__ __launch_bounds__(kThreads) void kv_attention_join_kernel(AttnArgs a) {
  constexpr int RT = 16 * CT;
  __shared__ f32x4_t part_o[kWaves][kWave];
  __shared__ float part_m[kWaves][kWave], part_l[kWaves][kWave];
  const int hk = blockIdx.x % a.Hk;
  const int chunk = *a.plan;
  Item it;
  if (!find_item<RT>(a, chunk, (blockIdx.z * gridDim.x + blockIdx.x) / a.Hk, true, it)) return;
  const Span sp = span_of<RT>(a, it);
  if (it.over || sp.chunks == 1 || it.slot + sp.chunks > a.max_slots) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n_cols = min(RT, it.rows * a.G - it.tile * RT);
  const float* ml = a.part + (size_t)a.max_slots * a.Hk * RT * D;
  const int per = (sp.chunks + kWaves - 1) / kWaves, n0 = wave * per, n1 = min(n0 + per, sp.chunks);
  const size_t step = (size_t)a.Hk * RT;
  for (int e0 = blockIdx.y * kWave; e0 < n_cols * (D / 4); e0 += gridDim.y * kWave) {
    const int c = (e0 + lane) / (D / 4), d = (e0 + lane - c * (D / 4)) * 4;  // c < RT: RT * D / 4 is a multiple of 64
    const size_t at = ((size_t)it.slot * a.Hk + hk) * RT + c;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int n = n0; n < n1; ++n) top = fmaxf(top, ml[(at + n * step) * 2]);
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int n = n0; n < n1; ++n) {
      const float mm = ml[(at + n * step) * 2];
      const float f = mm == -INFINITY ? 0.f : exp2_fast(mm - top);
      sum += f * ml[(at + n * step) * 2 + 1];
      o += f * *(const f32x4_t*)(a.part + (at + n * step) * D + d);
    }
    __syncthreads();  // the sums of the values before are read
    part_o[wave][lane] = o;
    part_m[wave][lane] = top;
    part_l[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || c >= n_cols) continue;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, part_m[w][lane]);
    sum = 0.f;
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mm = part_m[w][lane], f = mm == -INFINITY ? 0.f : exp2_fast(mm - top);
      sum += f * part_l[w][lane];
      o += f * part_o[w][lane];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int r = it.tile * RT + c, row = r / a.G, head = hk * a.G + (r - row * a.G);
    uint16_t b[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) b[x] = Qk<F16>::out(o[x] * inv);
    *(uint2*)((uint16_t*)a.out + (it.q0 + row) * a.o_st + head * a.o_sh + d) =
        make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
  }
}

// Tiles of 16 columns, by the mean columns of a request.
int col_tiles(int T, int B, int G, int D) {
  const int64_t rows = ((int64_t)T * G + B - 1) / B;
  if (rows <= 16) return 1;
  if (rows <= 32 || D > 256) return 2;
  return 4;
}

struct Grid {
  int ct, resident, max_tiles, max_slots, groups;
};

Grid grid_of(int T, int B, int Hq, int Hk, int D, int64_t tokens, int ct) {
  const int G = Hq / Hk;
  Grid r;
  r.ct = ct;
  const int RT = 16 * r.ct;
  const int64_t cols = (int64_t)T * G;
  // a request's last tile may be cut: ceil(rows * G / RT) tiles
  r.max_tiles = (int)(cols < cols / RT + B ? cols : cols / RT + B);
  r.resident = (workgroups_per_cu(D, r.ct) * 256 + Hk - 1) / Hk;
  // chunk >= total / (kRounds * resident), so the chunks of all tiles are at
  // most kRounds * resident and one more for each; of tiles that are cut (units >
  // chunk) there are at most total / chunk, and no more chunks than the longest table has
  const int64_t per_tile = (tokens / kUnit + 1 + kMinChunk - 1) / kMinChunk;
  const int64_t items = kRounds * (int64_t)r.resident + r.max_tiles;
  const int64_t slots = items < 2 * kRounds * (int64_t)r.resident ? items : 2 * kRounds * (int64_t)r.resident;
  const int64_t most = r.max_tiles * per_tile;
  r.max_slots = (int)(tokens <= kMinChunk * kUnit ? 0 : most < slots ? most : slots);
  // Workgroups without an item cost a round of the chip each time it is full of
  // them (2056 of them 9.6 us beside one request of 1391 tokens), so there are no
  // more than it holds at a time, or tiles; each takes every so-many-th item.
  const int64_t wide = r.resident > r.max_tiles ? r.resident : r.max_tiles;
  const int64_t groups = most < wide ? most : wide < items ? wide : items;
  r.groups = (int)(groups < kMaxGrid / Hk ? groups : kMaxGrid / Hk);
  return r;
}

// Bytes of the workspace in front of the partial sums.
size_t plan_bytes(int B) { return kEnds + (B > kWave ? ((size_t)B * sizeof(int4) + 63) / 64 * 64 : 0); }

size_t part_bytes(const Grid& gr, int B, int Hk, int D) {
  return plan_bytes(B) + (size_t)gr.max_slots * Hk * gr.ct * 16 * (D + 2) * sizeof(float);
}

bool width_ok(int D) { return D == 64 || D == 128 || D == 256 || D == 512; }

template <int D, int CT, bool F16>
void launch(const AttnArgs& a, const Grid& gr, hipStream_t stream) {
  if (a.B > kWave)
    hipLaunchKernelGGL(kv_attention_plan_kernel<16 * CT>, dim3(1), dim3(kPlanThreads), 0, stream, a);
  hipLaunchKernelGGL((kv_attention_kernel<D, CT, F16>), dim3(gr.groups * a.Hk), dim3(kThreads), 0, stream, a);
  // up to 2048 workgroups, each for as many of its tile's values as that leaves
  if (gr.max_slots == 0) return;
  const int cols = (int)min((int64_t)16 * CT, (int64_t)(a.q_start ? a.T : 1) * a.G);
  const int per = min(gr.max_tiles, kMaxGrid / a.Hk), layers = (gr.max_tiles - 1) / per + 1, tiles = per * a.Hk;
  const int parts = min(max(2048 / tiles, 1), (cols * (D / 4) + kWave - 1) / kWave);
  hipLaunchKernelGGL((kv_attention_join_kernel<D, CT, F16>), dim3(tiles, parts, layers), dim3(kThreads), 0, stream, a);
}

template <int D, bool F16>
void launch_ct(const AttnArgs& a, const Grid& gr, hipStream_t stream) {
  if (gr.ct == 1) launch<D, 1, F16>(a, gr, stream);
  else if (gr.ct == 2) launch<D, 2, F16>(a, gr, stream);
  else if constexpr (D <= 256) launch<D, 4, F16>(a, gr, stream);
}

template <bool F16>
void launch_d(const AttnArgs& a, const Grid& gr, int D, hipStream_t stream) {
  if (D == 64) launch_ct<64, F16>(a, gr, stream);
  else if (D == 128) launch_ct<128, F16>(a, gr, stream);
  else if (D == 256) launch_ct<256, F16>(a, gr, stream);
  else launch_ct<512, F16>(a, gr, stream);
}

}  // namespace

size_t kv_attention_workspace_bytes(int T, int B, int Hq, int Hk, int D, int64_t max_tokens) {
  if (T <= 0 || B <= 0 || Hk <= 0 || Hk > kMaxGrid || Hq <= 0 || Hq % Hk || !width_ok(D) || max_tokens < 0) return 0;
  // Fewer requests can mean wider tiles and more to hold: the most that any call of up to T rows and B
  // requests needs, width by width (the wider ones are of calls with few requests).
  const int64_t cols = (int64_t)T * (Hq / Hk);
  size_t need = 0;
  for (int ct = 1; ct <= col_tiles(T, 1, Hq / Hk, D); ct *= 2) {
    const int64_t most = ct == 1 ? B : (cols - 1) / (8 * ct);  // (cols + b - 1) / b > 8 ct
    const Grid gr = grid_of(T, (int)(most < B ? most : B), Hq, Hk, D, max_tokens, ct);
    const size_t bytes = part_bytes(gr, B, Hk, D);
    need = need > bytes ? need : bytes;
  }
  return need;
}

int launch_kv_attention(const void* q, int dtype, const int64_t* q_strides, const void* k_cache, const void* v_cache,
                        const float* k_scale, const float* v_scale, const int32_t* block_table, int64_t table_stride,
                        int max_pages, const int32_t* seq_lens, const int32_t* q_start, void* out,
                        const int64_t* o_strides, int T, int B, int Hq, int Hk, int D, int page_size,
                        int64_t num_pages, float scale, int window, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
  if (dtype != GI_DTYPE_BF16 && dtype != GI_DTYPE_FP16)
    return fail(GI_ERR_UNSUPPORTED, "kv_attention: query rows must be bf16 or fp16");
  if (T < 0 || B < 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || max_pages < 0 || table_stride < max_pages || num_pages < 0)
    return fail(GI_ERR_INVALID_ARG, "kv_attention: bad shape (Hq must be a multiple of Hk, table_stride >= max_pages)");
  if (!width_ok(D)) return fail(GI_ERR_UNSUPPORTED, "kv_attention: head widths 64, 128, 256 and 512");
  const int lp = log2_page(page_size);
  if (lp < 0) return fail(GI_ERR_INVALID_ARG, "kv_attention: page_size must be 16, 32, 64, 128 or 256");
  if (!q_start && T != B) return fail(GI_ERR_INVALID_ARG, "kv_attention: without q_start there is one row a request");
  if (Hk > kMaxGrid) return fail(GI_ERR_UNSUPPORTED, "kv_attention: at most 2^23 kv heads");
  if (B > kMaxRequests) return fail(GI_ERR_UNSUPPORTED, "kv_attention: at most 2^20 requests");
  if (!(scale == scale)) return fail(GI_ERR_INVALID_ARG, "kv_attention: scale is NaN");
  if (window < 0) return fail(GI_ERR_INVALID_ARG, "kv_attention: window must be >= 0 (0: none)");
  if ((int64_t)T * (Hq / Hk) > 0x3fffffff || (int64_t)max_pages * page_size > 0x3fffffff)
    return fail(GI_ERR_UNSUPPORTED, "kv_attention: too many rows, or a table of more than 2^30 tokens");
  if (T == 0 || B == 0) return GI_OK;
  if (num_pages == 0) return fail(GI_ERR_INVALID_ARG, "kv_attention: the cache has no pages");
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !seq_lens || !out || (max_pages > 0 && !block_table))
    return fail(GI_ERR_INVALID_ARG, "kv_attention: null pointer");
  for (const void* p : {q, k_cache, v_cache, (const void*)out})
    if (!aligned16(p)) return fail(GI_ERR_INVALID_ARG, "kv_attention: pointers must be 16-byte aligned");
  for (const int64_t s : {q_strides[0], q_strides[1], o_strides[0], o_strides[1]})
    if (s % 8) return fail(GI_ERR_INVALID_ARG, "kv_attention: row and head strides must be multiples of 8 elements");
  if (window >= (int64_t)max_pages * page_size) window = 0;  // no request is that long
  if (!aligned16(workspace)) return fail(GI_ERR_INVALID_ARG, "kv_attention: pointers must be 16-byte aligned");
  const Grid gr = grid_of(T, B, Hq, Hk, D, (int64_t)max_pages * page_size, col_tiles(T, B, Hq / Hk, D));
  if ((int64_t)gr.max_tiles * Hk > 0x7fffffff) return fail(GI_ERR_UNSUPPORTED, "kv_attention: too many rows");
  if (!workspace || workspace_bytes < part_bytes(gr, B, Hk, D))
    return fail(GI_ERR_WORKSPACE, "kv_attention: workspace missing or too small");
  AttnArgs a{q, q_strides[0], q_strides[1], (const uint8_t*)k_cache, (const uint8_t*)v_cache, k_scale, v_scale,
             block_table, table_stride, seq_lens, q_start, out, o_strides[0], o_strides[1], (int*)workspace,
             (float*)((char*)workspace + plan_bytes(B)),
             num_pages, scale * kLog2e, T, B, Hk, Hq / Hk, max_pages, lp, window, gr.resident, gr.max_slots};
  if (dtype == GI_DTYPE_FP16) launch_d<true>(a, gr, D, stream);
  else launch_d<false>(a, gr, D, stream);
  return after_launch("kv_attention launch");
}

}  // namespace gi
