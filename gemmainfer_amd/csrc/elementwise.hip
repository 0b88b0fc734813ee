// Companion kernels the drop-in module must export next to the MoE path:
// final-logit softcap, Gemma RMSNorm and rotate-half RoPE (gfx950).
//
// Reference behaviour restated (paths relative to the GemmaInfer repo):
//   softcap  csrc/softcapping.cu:7-19     x <- cap * tanh(x / cap)
//   rmsnorm  csrc/rmsnorm.cu:16-73         fp32 mean of squares, rsqrt(. + eps),
//                                          times weight or (1 + weight)
//   rope     csrc/rmsnorm.cu:116-164       x1' = x1 c1 - x2 s1, x2' = x2 c2 + x1 s2

#include "../../include/gemmainfer_amd.h"
#include "gi_common.h"
#include "gi_internal.h"

namespace gi {

namespace {

template <typename T>
__device__ __forceinline__ float ld(const T* p, int64_t i);
template <>
__device__ __forceinline__ float ld<uint16_t>(const uint16_t* p, int64_t i) {
  return bf16_to_f32(p[i]);
}
template <>
__device__ __forceinline__ float ld<_Float16>(const _Float16* p, int64_t i) {
  return (float)p[i];
}
template <>
__device__ __forceinline__ float ld<float>(const float* p, int64_t i) {
  return p[i];
}

__device__ __forceinline__ void st(uint16_t* p, int64_t i, float v) { p[i] = f32_to_bf16(v); }
__device__ __forceinline__ void st(_Float16* p, int64_t i, float v) { p[i] = (_Float16)v; }
__device__ __forceinline__ void st(float* p, int64_t i, float v) { p[i] = v; }

template <typename T>
__global__ __launch_bounds__(256) void softcap_kernel(T* x, int64_t n, float cap, float inv_cap) {
  const int64_t stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride)
    st(x, i, tanhf(ld(x, i) * inv_cap) * cap);
}

template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_kernel(const T* in, const T* w, T* out, int hidden,
                                                      float eps, int unit_offset) {
  __shared__ float partial[4];
  const int64_t row = blockIdx.x;
  const T* x = in + row * hidden;
  T* y = out + row * hidden;
  float ss = 0.f;
  for (int i = threadIdx.x; i < hidden; i += blockDim.x) {
    const float v = ld(x, i);
    ss += v * v;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, kWave);
  if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = ss;
  __syncthreads();
  const float total = partial[0] + partial[1] + partial[2] + partial[3];
  const float r = rsqrtf(total / (float)hidden + eps);
  for (int i = threadIdx.x; i < hidden; i += blockDim.x) {
    float v = ld(x, i) * r;
    if (w) {
      const float wv = ld(w, i);
      v *= unit_offset ? 1.f + wv : wv;
    }
    st(y, i, v);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void rope_kernel(T* q, T* k, const T* cs, const T* sn,
                                                   const int64_t* pos, int S, int Hq, int Hk,
                                                   int D, int64_t q_sb, int64_t q_sh,
                                                   int64_t q_ss, int64_t k_sb, int64_t k_sh,
                                                   int64_t k_ss) {
  const int bs = blockIdx.x, head = blockIdx.y;
  const int half = D >> 1;
  const int b = bs / S, s = bs - b * S;
  const int64_t p = pos[bs];
  T* base;
  if (head < Hq) base = q + b * q_sb + head * q_sh + s * q_ss;
  else base = k + b * k_sb + (head - Hq) * k_sh + s * k_ss;
  for (int d = threadIdx.x; d < half; d += blockDim.x) {
    const float c1 = ld(cs, p * D + d), s1 = ld(sn, p * D + d);
    const float c2 = ld(cs, p * D + d + half), s2 = ld(sn, p * D + d + half);
    const float x1 = ld(base, d), x2 = ld(base, d + half);
    st(base, d, x1 * c1 - x2 * s1);
    st(base, d + half, x2 * c2 + x1 * s2);
  }
}

// Rotary embedding of packed rows: the pair (x1, x2) of frequency f at position
// p becomes (x1 c - x2 s, x2 c + x1 s), c = m cos(p f), s = m sin(p f).  The
// angle is formed in fp64 and reduced to (-1/2, 1/2] turns before it is rounded
// to fp32: at a position of 10^6 an fp32 product would be off by up to 0.03
// radians, a reduced one by 1e-7.  A thread takes one unit (16 bytes, or a pair,
// of each half) of one head of one row; a workgroup the units of one row, whose cos and
// sin its threads work out once, into LDS, while their elements are on the way.  Bound by HBM: each
// element is read and written once.
constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 512;
constexpr int kRopeGrid = 1 << 23;  // rows along x: with a row's threads under the 2^32 that a launch may have

struct RopeArgs {
  const void* in[2];   // q, k
  void* out[2];
  int64_t in_st[2], in_sh[2], out_st[2], out_sh[2];  // row and head strides, elements
  const int64_t* pos;
  const double* freq;
  float mscale;
  int T, heads[2], D, pairs;
  int turn, units;     // units of a head that turn, and with those that are only copied
};

// Explicit fused steps, each rounded to fp32 (for fp16 results the compiler
// would otherwise join the last one and the conversion here and there): every
// form of the kernel gives the same bits.
__device__ __forceinline__ void turn_pair(float x1, float x2, float c, float s, float& y1, float& y2) {
  y1 = fmaf(x1, c, -(x2 * s));
  y2 = fmaf(x2, c, x1 * s);
  asm("" : "+v"(y1), "+v"(y2));
}

template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
  T v[N];
};

// kVec: units of 8 elements (rows, heads and the halves 16-byte aligned), 8
// pairs where the halves are apart and 4 where pairs are adjacent; otherwise a
// unit is a pair, or one element that is copied.
template <typename T, bool kInter, bool kVec>
__global__ __launch_bounds__(kRopeThreads) void rope_rows_kernel(RopeArgs a) {
  constexpr int N = kVec ? 8 : 1;
  __shared__ float cs[kRopeMaxPairs], sn[kRopeMaxPairs];
  const int64_t row = (int64_t)blockIdx.z * gridDim.x + blockIdx.x;
  if (row >= a.T) return;
  const int R = 2 * a.pairs;
  const int i = blockIdx.y * kRopeThreads + threadIdx.x;
  const int h = i / a.units, u = i - h * a.units;
  const bool on = h < a.heads[0] + a.heads[1], turns = u < a.turn;
  const int w = h < a.heads[0] ? 0 : 1, hw = h - (w ? a.heads[0] : 0);
  // the unit's elements: [d1, d1 + N) and, of a unit that turns and has its second half apart, [d2, d2 + N)
  const bool two = turns && (!kInter || !kVec);
  const int d1 = turns ? (kInter && !kVec ? 2 * u : u * N) : R + (u - a.turn) * N;
  const int d2 = kInter ? d1 + 1 : a.pairs + u * N;
  Pack<T, N> v1, v2;
  if (on) {
    const T* x = (const T*)a.in[w] + row * a.in_st[w] + hw * a.in_sh[w];
    v1 = *(const Pack<T, N>*)(x + d1);
    if (two) v2 = *(const Pack<T, N>*)(x + d2);
  }
  const double p = (double)a.pos[row];
  for (int j = threadIdx.x; j < a.pairs; j += kRopeThreads) {
    const double t = p * a.freq[j] * 0.15915494309189535;  // 1 / (2 pi)
    const float r = (float)(t - rint(t));
    float s, c;
    sincospif(2.f * r, &s, &c);
    cs[j] = c * a.mscale;
    sn[j] = s * a.mscale;
  }
  __syncthreads();
  if (!on) return;
  T* y = (T*)a.out[w] + row * a.out_st[w] + hw * a.out_sh[w];
  if (turns) {
    float y1, y2;
    if (two) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        turn_pair(ld(v1.v, j), ld(v2.v, j), cs[u * N + j], sn[u * N + j], y1, y2);
        st(v1.v, j, y1);
        st(v2.v, j, y2);
      }
      *(Pack<T, N>*)(y + d2) = v2;
    } else {
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        turn_pair(ld(v1.v, 2 * j), ld(v1.v, 2 * j + 1), cs[u * (N / 2) + j], sn[u * (N / 2) + j], y1, y2);
        st(v1.v, 2 * j, y1);
        st(v1.v, 2 * j + 1, y2);
      }
    }
  }
  *(Pack<T, N>*)(y + d1) = v1;
}

int check_dtype(int dt, const char* who) {
  if (dt != GI_DTYPE_BF16 && dt != GI_DTYPE_FP16 && dt != GI_DTYPE_FP32)
    return fail(GI_ERR_UNSUPPORTED, std::string(who) + ": dtype must be bf16, fp16 or fp32");
  return GI_OK;
}

}  // namespace

int launch_softcap(void* x, int dtype, int64_t n, float cap, hipStream_t stream) {
  int st = check_dtype(dtype, "softcap");
  if (st != GI_OK) return st;
  if (n < 0 || !(cap != 0.f)) return fail(GI_ERR_INVALID_ARG, "softcap: n >= 0 and cap != 0 required");
  if (n == 0) return GI_OK;
  if (!x) return fail(GI_ERR_INVALID_ARG, "softcap: null pointer");
  const int64_t want = (n + 255) / 256;
  const int blocks = (int)(want < 65536 ? want : 65536);
  const float inv = 1.0f / cap;
  if (dtype == GI_DTYPE_BF16)
    hipLaunchKernelGGL(softcap_kernel<uint16_t>, dim3(blocks), dim3(256), 0, stream, (uint16_t*)x, n, cap, inv);
  else if (dtype == GI_DTYPE_FP16)
    hipLaunchKernelGGL(softcap_kernel<_Float16>, dim3(blocks), dim3(256), 0, stream, (_Float16*)x, n, cap, inv);
  else
    hipLaunchKernelGGL(softcap_kernel<float>, dim3(blocks), dim3(256), 0, stream, (float*)x, n, cap, inv);
  return after_launch("softcap launch");
}

int launch_rmsnorm(const void* in, const void* weight, void* out, int dtype, int64_t rows,
                   int hidden, float eps, int add_unit_offset, hipStream_t stream) {
  int st = check_dtype(dtype, "rmsnorm");
  if (st != GI_OK) return st;
  if (rows < 0 || hidden <= 0) return fail(GI_ERR_INVALID_ARG, "rmsnorm: rows >= 0, hidden > 0 required");
  if (rows > 0x7fffffff) return fail(GI_ERR_UNSUPPORTED, "rmsnorm: too many rows");
  if (rows == 0) return GI_OK;
  if (!in || !out) return fail(GI_ERR_INVALID_ARG, "rmsnorm: null pointer");
  const dim3 grid((unsigned)rows);
  if (dtype == GI_DTYPE_BF16)
    hipLaunchKernelGGL(rmsnorm_kernel<uint16_t>, grid, dim3(256), 0, stream, (const uint16_t*)in,
                       (const uint16_t*)weight, (uint16_t*)out, hidden, eps, add_unit_offset);
  else if (dtype == GI_DTYPE_FP16)
    hipLaunchKernelGGL(rmsnorm_kernel<_Float16>, grid, dim3(256), 0, stream, (const _Float16*)in,
                       (const _Float16*)weight, (_Float16*)out, hidden, eps, add_unit_offset);
  else
    hipLaunchKernelGGL(rmsnorm_kernel<float>, grid, dim3(256), 0, stream, (const float*)in,
                       (const float*)weight, (float*)out, hidden, eps, add_unit_offset);
  return after_launch("rmsnorm launch");
}

int launch_rope(void* q, void* k, const void* cos_t, const void* sin_t, const int64_t* pos,
                int dtype, int B, int Hq, int Hk, int S, int D, const int64_t* qs,
                const int64_t* ks, hipStream_t stream) {
  int st = check_dtype(dtype, "rope");
  if (st != GI_OK) return st;
  if (B < 0 || Hq < 0 || Hk < 0 || S < 0 || D <= 0 || (D & 1))
    return fail(GI_ERR_INVALID_ARG, "rope: bad shape (D must be even and positive)");
  if (!k) Hk = 0;
  if (B == 0 || S == 0 || Hq + Hk == 0) return GI_OK;
  if (!q || !cos_t || !sin_t || !pos) return fail(GI_ERR_INVALID_ARG, "rope: null pointer");
  const dim3 grid((unsigned)(B * S), (unsigned)(Hq + Hk));
  const int threads = (D / 2) < 256 ? ((D / 2 + 63) / 64) * 64 : 256;
#define GI_ROPE(T)                                                                            \
  hipLaunchKernelGGL(rope_kernel<T>, grid, dim3(threads), 0, stream, (T*)q, (T*)k,          \
                     (const T*)cos_t, (const T*)sin_t, pos, S, Hq, Hk, D, qs[0], qs[1], qs[2], \
                     ks[0], ks[1], ks[2])
  if (dtype == GI_DTYPE_BF16) GI_ROPE(uint16_t);
  else if (dtype == GI_DTYPE_FP16) GI_ROPE(_Float16);
  else GI_ROPE(float);
#undef GI_ROPE
  return after_launch("rope launch");
}

int launch_rope_rows(const void* q, void* q_out, const void* k, void* k_out, const int64_t* positions,
                     const double* inv_freq, int dtype, int T, int Hq, int Hk, int D, int rotary_dim, int interleaved,
                     float mscale, const int64_t* q_strides, const int64_t* qo_strides, const int64_t* k_strides,
                     const int64_t* ko_strides, hipStream_t stream) {
  int st = check_dtype(dtype, "rope_rows");
  if (st != GI_OK) return st;
  if (T < 0 || Hq < 0 || Hk < 0 || D <= 0 || rotary_dim <= 0 || rotary_dim > D || (rotary_dim & 1))
    return fail(GI_ERR_INVALID_ARG, "rope_rows: T, Hq, Hk >= 0 and an even rotary_dim in [2, D] required");
  if (rotary_dim > 2 * kRopeMaxPairs) return fail(GI_ERR_UNSUPPORTED, "rope_rows: rotary_dim at most 1024");
  if (!k) Hk = 0;
  if (T == 0 || Hq + Hk == 0) return GI_OK;
  if ((Hq > 0 && (!q || !q_out)) || (Hk > 0 && !k_out) || !positions || !inv_freq)
    return fail(GI_ERR_INVALID_ARG, "rope_rows: null pointer");
  RopeArgs a{{q, k}, {q_out, k_out}, {q_strides[0], k_strides[0]}, {q_strides[1], k_strides[1]},
             {qo_strides[0], ko_strides[0]}, {qo_strides[1], ko_strides[1]}, positions, inv_freq, mscale, T, {Hq, Hk}, D,
             rotary_dim / 2, 0, 0};
  const int size = dtype == GI_DTYPE_FP32 ? 4 : 2;
  bool vec = D % 8 == 0 && rotary_dim % (interleaved ? 8 : 16) == 0;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    vec = vec && aligned16(a.in[w]) && aligned16(a.out[w]);
    for (const int64_t s : {a.in_st[w], a.in_sh[w], a.out_st[w], a.out_sh[w]}) vec = vec && s * size % 16 == 0;
  }
  // dimensions that do not turn are left alone where the result takes the place of the input
  const bool copy = (Hq > 0 && q != q_out) || (Hk > 0 && k != k_out);
  a.turn = !vec ? a.pairs : interleaved ? rotary_dim / 8 : rotary_dim / 16;
  a.units = a.turn + (copy ? (D - rotary_dim) / (vec ? 8 : 1) : 0);
  // (two units a thread, or a whole row in one workgroup: within 0.5 us for
  // 2047 rows of 16 + 8 heads of 256, 12.3 us)
  const int64_t parts = ((int64_t)(Hq + Hk) * a.units + kRopeThreads - 1) / kRopeThreads;
  if (parts > 65535) return fail(GI_ERR_UNSUPPORTED, "rope_rows: too many heads");
  const int width = T < kRopeGrid ? T : kRopeGrid;
  const dim3 grid(width, (unsigned)parts, (T - 1) / width + 1);
#define GI_ROPE_V(T_, I_)                                                                                 \
  do {                                                                                                    \
    if (vec) hipLaunchKernelGGL((rope_rows_kernel<T_, I_, true>), grid, dim3(kRopeThreads), 0, stream, a);  \
    else hipLaunchKernelGGL((rope_rows_kernel<T_, I_, false>), grid, dim3(kRopeThreads), 0, stream, a);     \
  } while (0)
#define GI_ROPE_I(T_)                 \
  do {                                \
    if (interleaved) GI_ROPE_V(T_, true); \
    else GI_ROPE_V(T_, false);        \
  } while (0)
  if (dtype == GI_DTYPE_BF16) GI_ROPE_I(uint16_t);
  else if (dtype == GI_DTYPE_FP16) GI_ROPE_I(_Float16);
  else GI_ROPE_I(float);
#undef GI_ROPE_I
#undef GI_ROPE_V
  return after_launch("rope_rows launch");
}

}  // namespace gi
