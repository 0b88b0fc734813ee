// The 8-bit paged K/V cache: where the rows of a step go (kv_slots) and how
// they are stored (kv_append).  kv_attention.hip reads it.
//
// Layout.  A page holds P rows (tokens) of every kv head as OCP e4m3 codes,
//   k_cache [pages, Hk, P, D]   a row's D codes together
//   v_cache [pages, Hk, D, P]   a dimension's P codes together
// and one fp32 scale per (page, head) for K and one for V: value = code *
// scale.  V is held transposed because the matrix cores contract P.V over
// rows: a lane then reads 16 rows of its dimension with one 16-byte load, where
// [P, D] would need a transposition in registers or LDS for every page on every
// decode step.  The price is paid once per row, at append: a lone row's V codes
// are single bytes P apart.
//
// Scales are powers of two, the smallest that brings the page's largest value
// under 448 (the largest e4m3).  With those, x / scale is exact, a stored value
// code * scale is exact in bf16 and fp32, and when a larger row arrives the
// page's codes move to the larger scale by a change of exponent (rounded only
// where they fall under e4m3's smallest normal number).

#include <numeric>
#include <type_traits>

#include "../../include/gemmainfer_amd.h"
#include "gi_common.h"
#include "gi_internal.h"

namespace gi {

namespace {

// ---------------------------------------------------------------------------
// kv_slots
// ---------------------------------------------------------------------------
// One launch, no exchange between workgroups: each scans the B request lengths
// into its own LDS (8 bytes of global reads a request) and then places its
// 256 tokens (7 requests 3.4 us, 301 requests and 14,500 rows 5.5 us).  A fresh
// page j of a request starts at position j*P >= ctx, which is one of the call's
// own tokens: that token's thread writes the table entry, so table entries are
// never read and written in one call.  Bound by latency
// (lengths -> scan -> table entry -> slot).
constexpr int kSlotThreads = 256;
constexpr int kMaxRequests = 8192;  // two ints a request in LDS: 64 KB

struct SlotArgs {
  const int32_t* ctx;
  const int32_t* add;
  int32_t* table;
  const int32_t* free_pages;
  const int32_t* used;
  int64_t* slots;
  int64_t* positions;
  int32_t* q_start;
  int32_t* seq_lens;
  int32_t* status;
  int64_t table_stride;
  int B, cols, n_free, log_page, n;
};

// Inclusive scan over the workgroup; `total` gets the sum.  Two barriers.
template <typename I>
__device__ __forceinline__ I block_scan(I v, I* part, I& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const I u = __shfl_up(v, off, kWave);
    if (lane >= off) v += u;
  }
  __syncthreads();  // the previous scan's readers are done with `part`
  if (lane == 63) part[wave] = v;
  __syncthreads();
  I before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSlotThreads / kWave; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return v + before;
}

__global__ __launch_bounds__(kSlotThreads) void kv_slots_kernel(SlotArgs a) {
  extern __shared__ int lds[];
  int* start = lds;         // [B] first row of each request, at most n
  int* fresh = lds + a.B;   // [B] fresh pages of the requests before it
  __shared__ long long part64[kSlotThreads / kWave];
  __shared__ int part32[kSlotThreads / kWave];
  const int tid = threadIdx.x;
  const int up = (1 << a.log_page) - 1;
  long long rows = 0, lack = 0;  // rows asked for so far; pages behind the table's last column
  int pages = 0;
  for (int b0 = 0; b0 < a.B; b0 += kSlotThreads) {
    const int b = b0 + tid;
    const bool on = b < a.B;
    const long long ctx = on ? max(a.ctx[b], 0) : 0;
    const long long add = on ? max(a.add[b], 0) : 0;
    long long sum;
    const long long end = rows + block_scan<long long>(add, part64, sum);
    rows += sum;
    const long long first = min(end - add, (long long)a.n);
    const long long len = ctx + min(add, (long long)a.n - first);
    const long long have = (ctx + up) >> a.log_page, want = (len + up) >> a.log_page;
    const int count = (int)(min(want, (long long)a.cols) - min(have, (long long)a.cols));
    lack += want - have - count;
    int psum;
    const int pend = pages + block_scan<int>(count, part32, psum);
    pages += psum;
    if (on) {
      start[b] = (int)first;
      fresh[b] = pend - count;
      if (blockIdx.x == 0) {
        a.q_start[b] = (int)first;
        a.seq_lens[b] = (int)min(len, 0x7fffffffLL);
      }
    }
  }
  const int live = (int)min(rows, (long long)a.n);
  const int used = max(a.used[0], 0);
  if (blockIdx.x == 0) {
    long long all;
    block_scan<long long>(lack, part64, all);
    if (tid == 0) {
      const int got = min(pages, max(a.n_free - used, 0));
      a.q_start[a.B] = live;
      a.status[0] = used + got;
      a.status[1] = (int)min(all + pages - got, 0x7fffffffLL);
      a.status[2] = (int)min(rows - live, 0x7fffffffLL);
    }
  }
  __syncthreads();
  const int t = blockIdx.x * kSlotThreads + tid;
  if (t >= a.n) return;
  long long slot = -1, pos = 0;
  if (t < live) {
    int lo = 0, hi = a.B - 1;  // the last request whose first row is at most t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    const long long ctx = max(a.ctx[lo], 0);
    pos = ctx + (t - start[lo]);
    const long long j = pos >> a.log_page, have = (ctx + up) >> a.log_page;
    if (j < a.cols) {
      int32_t* entry = a.table + lo * a.table_stride + j;
      long long page;
      if (j < have) {
        page = *entry;
      } else {
        const long long at = (long long)used + fresh[lo] + (j - have);
        page = at < a.n_free ? a.free_pages[at] : -1;
        if ((pos & up) == 0) *entry = (int)page;
      }
      if (page >= 0) slot = (page << a.log_page) + (pos & up);
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

// ---------------------------------------------------------------------------
// kv_append
// ---------------------------------------------------------------------------
constexpr int kAppThreads = 256;
constexpr int kMaxPage = 256;
// slots a lane loads at a time where it looks for a run's start or end over skipped rows (with eight the
// kernel takes 92 registers instead of 76: 1024 decoded rows 47 us, with four 42)
constexpr int kLookRows = 4;
constexpr uint32_t kAppGrid = 1u << 23;  // workgroups along x: with their threads under the 2^32 that a launch may have

struct AppendArgs {
  const void* x[2];        // K rows, V rows
  int64_t st[2], sh[2];    // row and head strides, elements
  const int64_t* slots;
  uint8_t* cache[2];
  float* scale[2];
  int64_t num_pages;
  int T, Hk, D, log_page, per_wg;
  uint32_t blocks, spread;  // workgroup i of `blocks` looks at rows (i * spread mod blocks) * per_wg ...
};

template <typename T>
struct Vec8;  // eight consecutive elements as floats
template <>
struct Vec8<uint16_t> {
  static __device__ __forceinline__ void load(const uint16_t* p, float* f) {
    const uint4 d = *(const uint4*)p;
    const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf16lo(w[i]);
      f[2 * i + 1] = bf16hi(w[i]);
    }
  }
  static __device__ __forceinline__ float one(const uint16_t* p) { return bf16_to_f32(*p); }
};
template <>
struct Vec8<_Float16> {
  static __device__ __forceinline__ void load(const _Float16* p, float* f) {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 d = *(const h8*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)d[i];
  }
  static __device__ __forceinline__ float one(const _Float16* p) { return (float)*p; }
};
template <>
struct Vec8<float> {
  static __device__ __forceinline__ void load(const float* p, float* f) {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};

template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* p, float* f) {
  if (kVec) {
    Vec8<T>::load(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Vec8<T>::one(p + i);
  }
}

// e4m3 codes of four values (round to nearest even; |f| <= 448).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}

// The codes of `w` for a scale 1/ratio times the old one.
__device__ __forceinline__ uint32_t rescale_e4m3(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return pack_e4m3(lo[0] * ratio, lo[1] * ratio, hi[0] * ratio, hi[1] * ratio);
}

// The smallest power of two s in [2^-40, 2^40] with amax <= 448 s (448 = 1.75 *
// 2^8), from amax's bits; NaN where there is none (amax infinite, NaN or larger).
__device__ __forceinline__ float page_scale(uint32_t amax_bits) {
  int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (e > 40) return __uint_as_float(0x7fc00000u);
  e = max(e, -40);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// One workgroup a (run of rows, head, K or V); a run is the rows of the call
// that follow each other on one page, rows that are skipped between them or not,
// and its first row's workgroup does it all: which row lands on each of the
// page's P places (the last one wins where a slot is named twice), the largest
// value of those rows, the page's scale, then the codes.  Everything of a page in
// one workgroup needs no atomics on scales and no second launch.  A decode step
// is bound by latency (slots, then rows and scale, then stores: 61 rows of 8 heads
// of 256 in 6 us), a prompt by its rows' two reads (6000 rows: 27 to 29 us, 74 MB
// in and out; kept in registers instead, fewer workgroups fit and it takes 34).
// per_wg rows are looked at by one workgroup.
template <typename T, bool kVec>
__global__ __launch_bounds__(kAppThreads) void kv_append_kernel(AppendArgs a) {
  __shared__ int last[kMaxPage];               // the row on each place, -1: none
  __shared__ int place[kMaxPage];              // the places that have one
  __shared__ uint32_t group_rows[kMaxPage / 16];  // ... as bits of each 16 places
  __shared__ uint32_t wave_max[kAppThreads / kWave];
  __shared__ int wave_end[kAppThreads / kWave], wave_count[kAppThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, head = blockIdx.y, kv = blockIdx.z & 1;
  const uint32_t block = (blockIdx.z >> 1) * gridDim.x + blockIdx.x;
  if (block >= a.blocks) return;
  const int lp = a.log_page, P = 1 << lp, D = a.D;
  const T* x = (const T*)a.x[kv] + head * a.sh[kv];
  const int64_t st = a.st[kv];
  const int t_first = (int)(block * a.spread % a.blocks) * a.per_wg;
  auto on_page = [&](int64_t s) { return s >= 0 && s >> lp < a.num_pages; };
  // the first rows of runs among this workgroup's rows (every wave finds them
  // all): those whose page is not that of the last row before them that has one.
  // Lanes 0 ... back - 1 look at the rows in front of the workgroup's own.
  const int back = kWave - a.per_wg, t_look = t_first - back;
  unsigned long long runs;
  {
    const int t = t_look + lane;
    const int64_t s = t >= 0 && t < a.T ? a.slots[t] : -1;
    const bool ok = on_page(s);
    const unsigned long long oks = __ballot(ok), below = oks & ((1ull << lane) - 1);
    const long long page = s >> lp, before = __shfl(page, below ? 63 - __clzll(below) : lane, kWave);
    runs = __ballot(ok && lane >= back && (!below || before != page));
    const int first = oks ? __ffsll(oks) - 1 : 0;
    if (first >= back && runs) {
      // nothing but skipped rows in sight of it: further back, 256 rows at a time
      const long long its = __shfl(page, first, kWave);
      bool found = false;
      for (int end = t_look; end > 0 && !found; end -= kLookRows * kWave) {
        int64_t p[kLookRows];
#pragma unroll
        for (int i = 0; i < kLookRows; ++i) p[i] = end - 1 - i * kWave - lane >= 0 ? a.slots[end - 1 - i * kWave - lane] : -1;
#pragma unroll
        for (int i = 0; i < kLookRows; ++i) {
          const unsigned long long hit = __ballot(on_page(p[i]));
          if (found || !hit) continue;
          found = true;
          if (__shfl((long long)(p[i] >> lp), __ffsll(hit) - 1, kWave) == its) runs &= ~(1ull << first);
        }
      }
    }
  }
  for (; runs; runs &= runs - 1) {
    const int t0 = t_look + __ffsll(runs) - 1;
    const int64_t page = a.slots[t0] >> lp;
    float* scale = a.scale[kv] + page * a.Hk + head;
    const float old = *scale;
    __syncthreads();  // the run before is done with LDS
    if (tid < P) last[tid] = -1;
    // ---- the run's rows: those on the page up to the first one of another page
    auto look = [&](int base, auto count) {  // at `count` rows a thread; true where the run ends
      constexpr int kRows = decltype(count)::value;
      int64_t s[kRows];
      int end = 0x7fffffff;
#pragma unroll
      for (int i = 0; i < kRows; ++i) s[i] = base + i * kAppThreads + tid < a.T ? a.slots[base + i * kAppThreads + tid] : -1;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const unsigned long long other = __ballot(on_page(s[i]) && s[i] >> lp != page);
        if (other) end = min(end, base + i * kAppThreads + wave * kWave + __ffsll(other) - 1);
      }
      if (lane == 0) wave_end[wave] = end;
      __syncthreads();
      end = min(min(wave_end[0], wave_end[1]), min(wave_end[2], wave_end[3]));
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int t = base + i * kAppThreads + tid;
        if (t < end && s[i] >= 0 && s[i] >> lp == page) atomicMax(&last[s[i] & (P - 1)], t);
      }
      __syncthreads();
      return end != 0x7fffffff || base + kRows * kAppThreads >= a.T;
    };
    if (!look(t0, std::integral_constant<int, 1>()))
      for (int base = t0 + kAppThreads; !look(base, std::integral_constant<int, kLookRows>()); base += kLookRows * kAppThreads) {
      }
    const bool on = tid < P && last[tid] >= 0;
    const unsigned long long bits = __ballot(on);
    if (lane < 4 && wave * 4 + lane < P >> 4) group_rows[wave * 4 + lane] = (uint32_t)(bits >> (16 * lane)) & 0xffffu;
    if (lane == 0) wave_count[wave] = __popcll(bits);
    __syncthreads();
    int at = __popcll(bits & ((1ull << lane) - 1)), n = 0;
#pragma unroll
    for (int w = 0; w < kAppThreads / kWave; ++w) {
      at += w < wave ? wave_count[w] : 0;
      n += wave_count[w];
    }
    if (on) place[at] = tid;
    __syncthreads();
    // ---- their largest value
    const int per_row = D >> 3;  // threads of 8 elements
    uint32_t m = 0;
#pragma unroll 4
    for (int i = tid; i < n * per_row; i += kAppThreads) {
      const int r = i / per_row, c = (i - r * per_row) << 3;
      float f[8];
      load8<T, kVec>(x + last[place[r]] * st + c, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, kWave));
    if (lane == 0) wave_max[wave] = m;
    __syncthreads();
    m = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
    const float need = page_scale(m);
    const bool restart = last[0] >= 0;
    float now = need;
    if (!restart && !(old < need)) now = need == need ? old : need;  // old >= need, or one of them NaN
    if (tid == 0) *scale = now;
    const bool valid = now == now;
    const float inv = valid ? 1.f / now : 0.f;                       // a page without a scale holds zeros
    const bool move = !restart && valid && now > old;
    const float ratio = move ? old * inv : 1.f;
    uint8_t* codes = a.cache[kv] + (page * a.Hk + head) * ((int64_t)D << lp);
    if (kv == 0) {
#pragma unroll 4
      for (int i = tid; i < n * per_row; i += kAppThreads) {
        const int r = i / per_row, c = (i - r * per_row) << 3, p = place[r];
        float f[8];
        load8<T, kVec>(x + last[p] * st + c, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = valid ? f[j] * inv : 0.f;
        *(uint2*)(codes + (int64_t)p * D + c) =
            make_uint2(pack_e4m3(f[0], f[1], f[2], f[3]), pack_e4m3(f[4], f[5], f[6], f[7]));
      }
      if (move) {
        for (int i = tid; i < P * per_row; i += kAppThreads) {
          const int p = i / per_row, c = (i - p * per_row) << 3;
          if (last[p] >= 0) continue;
          uint2* dst = (uint2*)(codes + (int64_t)p * D + c);
          const uint2 w = *dst;
          *dst = make_uint2(rescale_e4m3(w.x, ratio), rescale_e4m3(w.y, ratio));
        }
      }
    } else {
      // a thread takes one dimension of 16 places: its codes are 16 adjacent bytes
      for (int i = tid; i < D * (P >> 4); i += kAppThreads) {
        const int g = i / D, d = i - g * D;
        const uint32_t rows = group_rows[g];
        if (rows == 0 && !move) continue;
        uint8_t* dst = codes + ((int64_t)d << lp) + g * 16;
        if (rows == 0xffffu || move) {
          float f[16];
#pragma unroll
          for (int p = 0; p < 16; ++p) f[p] = Vec8<T>::one(x + max(last[g * 16 + p], t0) * st + d);  // t0: any row
          uint32_t o[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int y = 0; y < 4; ++y) f[4 * q + y] = valid ? f[4 * q + y] * inv : 0.f;
            // a value of no place could be out of range: keep it from the conversion
#pragma unroll
            for (int y = 0; y < 4; ++y) f[4 * q + y] = rows >> (4 * q + y) & 1 ? f[4 * q + y] : 0.f;
            o[q] = pack_e4m3(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
          }
          if (rows != 0xffffu) {
            const uint4 w = *(const uint4*)dst;
            const uint32_t h[4] = {rescale_e4m3(w.x, ratio), rescale_e4m3(w.y, ratio), rescale_e4m3(w.z, ratio),
                                   rescale_e4m3(w.w, ratio)};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t b = rows >> (4 * q) & 0xfu;
              const uint32_t keep = (b & 1 ? 0xffu : 0u) | (b & 2 ? 0xff00u : 0u) | (b & 4 ? 0xff0000u : 0u) |
                                    (b & 8 ? 0xff000000u : 0u);
              o[q] = (o[q] & keep) | (h[q] & ~keep);
            }
          }
          *(uint4*)dst = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
          for (uint32_t left = rows; left; left &= left - 1) {
            const int p = __ffs((int)left) - 1;
            const float f = valid ? Vec8<T>::one(x + last[g * 16 + p] * st + d) * inv : 0.f;
            dst[p] = (uint8_t)pack_e4m3(f, 0.f, 0.f, 0.f);
          }
        }
      }
    }
  }
}

}  // namespace

int launch_kv_slots(const int32_t* ctx_lens, const int32_t* new_lens, int B, int32_t* block_table, int max_pages,
                    int64_t table_stride, const int32_t* free_pages, int n_free, const int32_t* free_used,
                    int page_size, int64_t* slots, int64_t* positions, int n_tokens, int32_t* q_start,
                    int32_t* seq_lens, int32_t* status, hipStream_t stream) {
  if (B < 0 || max_pages < 0 || n_free < 0 || n_tokens < 0 || table_stride < max_pages)
    return fail(GI_ERR_INVALID_ARG, "kv_slots: negative size, or table_stride < max_pages");
  if (B > kMaxRequests) return fail(GI_ERR_UNSUPPORTED, "kv_slots: at most 8192 requests");
  const int lp = log2_page(page_size);
  if (lp < 0) return fail(GI_ERR_INVALID_ARG, "kv_slots: page_size must be 16, 32, 64, 128 or 256");
  if (!free_used || !q_start || !status || (n_free > 0 && !free_pages) || (n_tokens > 0 && (!slots || !positions)) ||
      (B > 0 && (!ctx_lens || !new_lens || !seq_lens || (max_pages > 0 && !block_table))))
    return fail(GI_ERR_INVALID_ARG, "kv_slots: null pointer");
  SlotArgs a{ctx_lens, new_lens, block_table, free_pages, free_used, slots,  positions, q_start,
             seq_lens, status,   table_stride, B,         max_pages, n_free, lp,        n_tokens};
  const int wgs = n_tokens > 0 ? (n_tokens - 1) / kSlotThreads + 1 : 1;
  hipLaunchKernelGGL(kv_slots_kernel, dim3(wgs), dim3(kSlotThreads), (size_t)B * 2 * sizeof(int), stream, a);
  return after_launch("kv_slots launch");
}

int launch_kv_append(const void* k, const void* v, int dtype, const int64_t* k_strides, const int64_t* v_strides,
                     const int64_t* slots, int T, int Hk, int D, int page_size, int64_t num_pages, void* k_cache,
                     void* v_cache, float* k_scale, float* v_scale, hipStream_t stream) {
  if (dtype != GI_DTYPE_BF16 && dtype != GI_DTYPE_FP16 && dtype != GI_DTYPE_FP32)
    return fail(GI_ERR_UNSUPPORTED, "kv_append: rows must be bf16, fp16 or fp32");
  const int lp = log2_page(page_size);
  if (lp < 0) return fail(GI_ERR_INVALID_ARG, "kv_append: page_size must be 16, 32, 64, 128 or 256");
  if (T < 0 || Hk <= 0 || num_pages < 0 || D <= 0 || D % 8 || D > 1024)
    return fail(GI_ERR_INVALID_ARG, "kv_append: T, num_pages >= 0, Hk > 0 and D a multiple of 8 up to 1024 required");
  if (Hk > 65535) return fail(GI_ERR_UNSUPPORTED, "kv_append: at most 65535 kv heads");
  if (T > 1 << 30) return fail(GI_ERR_UNSUPPORTED, "kv_append: at most 2^30 rows");
  if (T == 0 || num_pages == 0) return GI_OK;
  if (!k || !v || !slots || !k_cache || !v_cache || !k_scale || !v_scale)
    return fail(GI_ERR_INVALID_ARG, "kv_append: null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache))
    return fail(GI_ERR_INVALID_ARG, "kv_append: the cache must be 16-byte aligned");
  AppendArgs a{};
  a.x[0] = k;
  a.x[1] = v;
  a.st[0] = k_strides[0];
  a.sh[0] = k_strides[1];
  a.st[1] = v_strides[0];
  a.sh[1] = v_strides[1];
  a.slots = slots;
  a.cache[0] = (uint8_t*)k_cache;
  a.cache[1] = (uint8_t*)v_cache;
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.num_pages = num_pages;
  a.T = T;
  a.Hk = Hk;
  a.D = D;
  a.log_page = lp;
  // a decode step's rows lie on pages of their own: a workgroup each; a
  // prompt's lie on its pages in runs, and most workgroups would find nothing.
  // The host sees only how many rows there are.  8 heads of 256, with 16, 4 and 1
  // rows a workgroup: 1200 prompt rows 14, 18 and 32 us, 6000 28, 47 and 141; of
  // lone rows 1040 48, 39 and 44, 2000 83, 67 and 79.
  a.per_wg = (int64_t)T * Hk > 8192 ? 16 : 1;
  // Of a prompt's workgroups every (page / 16)-th finds a run: in order, those
  // would all fall on a few of the chip's eight parts (6000 rows onto pages of
  // 64: 29.7 us, spread out 28.5).
  const uint32_t blocks = (uint32_t)((T - 1) / a.per_wg + 1);
  a.blocks = blocks;
  a.spread = 1;
  if (a.per_wg > 1 && blocks < 1u << 25) {
    a.spread = 61;
    while (std::gcd(a.spread, blocks) != 1) ++a.spread;  // one of a few: at most 25 bits of primes divide `blocks`
  }
  const int size = dtype == GI_DTYPE_FP32 ? 4 : 2;
  bool vec = aligned16(k) && aligned16(v);
  for (int i = 0; i < 2; ++i) vec = vec && a.st[i] * size % 16 == 0 && a.sh[i] * size % 16 == 0;
  const uint32_t width = blocks < kAppGrid ? blocks : kAppGrid;
  const dim3 grid(width, Hk, 2 * ((blocks - 1) / width + 1));
#define GI_APPEND(T_)                                                                                        \
  do {                                                                                                       \
    if (vec) hipLaunchKernelGGL((kv_append_kernel<T_, true>), grid, dim3(kAppThreads), 0, stream, a);        \
    else hipLaunchKernelGGL((kv_append_kernel<T_, false>), grid, dim3(kAppThreads), 0, stream, a);           \
  } while (0)
  if (dtype == GI_DTYPE_BF16) GI_APPEND(uint16_t);
  else if (dtype == GI_DTYPE_FP16) GI_APPEND(_Float16);
  else GI_APPEND(float);
#undef GI_APPEND
  return after_launch("kv_append launch");
}

}  // namespace gi
