// Global gradient norm over many tensors, clipping, and the clipped SGD step of
// fp32 masters, for MI355X (gfx950).
//
//   norm  = sqrt(sum_i |g_i|^2)      scale = min(1, max_norm / (norm + eps))
//   step:  u = scale * g + wd * m;  [b = mu * b + u; u = b;]  m -= lr * u;  p = bf16(m)
//
// Many tensors in one launch: their addresses and lengths ride in the kernel's
// arguments (no table to copy, so a call can be captured), a block walks chunks
// of CLIP_CHUNK elements over all of them. Each thread squares and adds a chunk
// in fp32, chunks and blocks add in fp64 in a fixed order: no atomics, the same
// gradients always give the same norm. Bound by HBM: the gradients are read once
// for the norm and once where they are scaled or applied. Four tensors of 67 million: the norm
// 190 us in fp32 (5.7 TB/s) and 94 in bf16, scaling in place 437 (4.9 TB/s) and 203.
#include "common.h"

#define CLIP_TENSORS 64
#define CLIP_CHUNK 16384
#define CLIP_BLOCKS 2048
enum { CLIP_BF16 = 0, CLIP_F16 = 1, CLIP_F32 = 2 };

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

struct ClipTensors {
  void* p[CLIP_TENSORS];
  long n[CLIP_TENSORS];
  int first[CLIP_TENSORS + 1];  // first chunk of each
  unsigned char kind[CLIP_TENSORS];
  int count;
};

struct StepTensors {
  __bf16* p[CLIP_TENSORS];
  float* m[CLIP_TENSORS];
  const void* g[CLIP_TENSORS];
  float* b[CLIP_TENSORS];
  long n[CLIP_TENSORS];
  int first[CLIP_TENSORS + 1];
  unsigned char kind[CLIP_TENSORS];
  int count;
};

// the tensor of a chunk: the last one that starts at or before it
template <typename A>
LAH_DEVINL int tensor_of(const A& a, int chunk) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int KIND>
LAH_DEVINL float load_one(const void* p, long i) {
  if (KIND == CLIP_BF16) return bf2f(((const __bf16*)p)[i]);
  if (KIND == CLIP_F16) return (float)((const _Float16*)p)[i];
  return ((const float*)p)[i];
}

template <int KIND>
LAH_DEVINL void load8(const void* p, long i, float (&v)[8]) {
  if (KIND == CLIP_F32) {
    *(f32x4*)v = *(const f32x4*)((const float*)p + i);
    *(f32x4*)(v + 4) = *(const f32x4*)((const float*)p + i + 4);
  } else if (KIND == CLIP_BF16) {
    const bf16x8 x = *(const bf16x8*)((const __bf16*)p + i);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = bf2f(x[q]);
  } else {
    const f16x8 x = *(const f16x8*)((const _Float16*)p + i);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = (float)x[q];
  }
}

LAH_DEVINL bool aligned16(const void* p) { return ((unsigned long long)p & 15) == 0; }

// a thread's squares in a chunk, added in T
template <int KIND, typename T>
LAH_DEVINL T chunk_squares(const void* p, long from, long to) {
  T s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (aligned16(p) && to - from == CLIP_CHUNK) {
#pragma unroll
    for (int i = 0; i < CLIP_CHUNK / 2048; ++i) {
      float v[8];
      load8<KIND>(p, from + i * 2048 + threadIdx.x * 8, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) s[q] += (T)v[q] * (T)v[q];
    }
  } else {
    for (long i = from + threadIdx.x; i < to; i += 256) {
      const T v = (T)load_one<KIND>(p, i);
      s[0] += v * v;
    }
  }
  return ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

// In fp32; where finite gradients of 2^64 and more leave its range, again in fp64.
template <int KIND>
LAH_DEVINL double squares_of(const void* p, long from, long to) {
  const float s = chunk_squares<KIND, float>(p, from, to);
  return isinf(s) ? chunk_squares<KIND, double>(p, from, to) : (double)s;
}

LAH_DEVINL double block_sum(double v, double* lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  const int waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
  for (int w = 0; w < waves; ++w) s += lds[w];
  return s;
}

__launch_bounds__(256) __global__ void clip_squares_kernel(ClipTensors a, double* __restrict__ partial) {
  __shared__ double lds[4];
  double sum = 0;
  for (int c = blockIdx.x; c < a.first[a.count]; c += gridDim.x) {
    const int t = tensor_of(a, c);
    const long from = (long)(c - a.first[t]) * CLIP_CHUNK, to = min(from + CLIP_CHUNK, a.n[t]);
    if (a.kind[t] == CLIP_F32) sum += squares_of<CLIP_F32>(a.p[t], from, to);
    else if (a.kind[t] == CLIP_BF16) sum += squares_of<CLIP_BF16>(a.p[t], from, to);
    else sum += squares_of<CLIP_F16>(a.p[t], from, to);
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// norm and scale from all blocks' sums; not-a-number stays one in both
__launch_bounds__(1024) __global__ void clip_finish_kernel(const double* __restrict__ partial, int n,
                                                           float max_norm, float eps,
                                                           float* __restrict__ norm,
                                                           float* __restrict__ scale) {
  __shared__ double lds[16];
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
  s = block_sum(s, lds);
  if (threadIdx.x == 0) {
    const double root = sqrt(s), c = (double)max_norm / (root + (double)eps);
    *norm = (float)root;
    *scale = c >= 1.0 ? 1.0f : (float)c;
  }
}

template <typename T8, typename T>
LAH_DEVINL void chunk_scale(T* p, long from, long to, float s) {
  if (aligned16(p) && to - from == CLIP_CHUNK) {
    for (int i = 0; i < CLIP_CHUNK / 2048; ++i) {
      T8* at = (T8*)(p + from + i * 2048 + threadIdx.x * 8);
      T8 x = *at;
#pragma unroll
      for (int q = 0; q < 8; ++q) x[q] = (T)((float)x[q] * s);
      *at = x;
    }
  } else {
    for (long i = from + threadIdx.x; i < to; i += 256) p[i] = (T)((float)p[i] * s);
  }
}

typedef __attribute__((ext_vector_type(8))) float f32x8;

// g *= scale in place; a scale of exactly 1 leaves every bit, so nothing is touched
__launch_bounds__(256) __global__ void clip_scale_kernel(ClipTensors a, const float* __restrict__ scale) {
  const float s = *scale;
  if (s == 1.0f) return;
  for (int c = blockIdx.x; c < a.first[a.count]; c += gridDim.x) {
    const int t = tensor_of(a, c);
    const long from = (long)(c - a.first[t]) * CLIP_CHUNK, to = min(from + CLIP_CHUNK, a.n[t]);
    if (a.kind[t] == CLIP_F32) chunk_scale<f32x8>((float*)a.p[t], from, to, s);
    else if (a.kind[t] == CLIP_BF16) chunk_scale<bf16x8>((__bf16*)a.p[t], from, to, s);
    else chunk_scale<f16x8>((_Float16*)a.p[t], from, to, s);
  }
}

template <int KIND, bool MOM>
LAH_DEVINL void chunk_step(const StepTensors& a, int t, long from, long to, float s, float lr, float mu,
                           float wd) {
  __bf16* p = a.p[t];
  float *m = a.m[t], *b = a.b[t];
  const void* g = a.g[t];
  const bool wide = aligned16(p) && aligned16(m) && aligned16(g) && (!MOM || aligned16(b));
  long i = from;
  if (wide) {
    for (; i + 2048 <= to; i += 2048) {
      const long at = i + threadIdx.x * 8;
      float gv[8], mv[8], bv[8];
      load8<KIND>(g, at, gv);
      load8<CLIP_F32>(m, at, mv);
      if (MOM) load8<CLIP_F32>(b, at, bv);
      bf16x8 o;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float u = gv[q] * s + wd * mv[q];
        if (MOM) u = bv[q] = mu * bv[q] + u;
        mv[q] -= lr * u;
        o[q] = f2bf(mv[q]);
      }
      *(f32x4*)(m + at) = *(f32x4*)mv;
      *(f32x4*)(m + at + 4) = *(f32x4*)(mv + 4);
      if (MOM) {
        *(f32x4*)(b + at) = *(f32x4*)bv;
        *(f32x4*)(b + at + 4) = *(f32x4*)(bv + 4);
      }
      *(bf16x8*)(p + at) = o;
    }
  }
  for (i += threadIdx.x; i < to; i += 256) {
    float u = load_one<KIND>(g, i) * s + wd * m[i];
    if (MOM) u = b[i] = mu * b[i] + u;
    const float v = m[i] - lr * u;
    m[i] = v;
    p[i] = f2bf(v);
  }
}

template <bool MOM>
__launch_bounds__(256) __global__ void master_sgd_kernel(StepTensors a, const float* __restrict__ scale,
                                                         float lr, float mu, float wd) {
  const float s = scale != nullptr ? *scale : 1.0f;
  for (int c = blockIdx.x; c < a.first[a.count]; c += gridDim.x) {
    const int t = tensor_of(a, c);
    const long from = (long)(c - a.first[t]) * CLIP_CHUNK, to = min(from + CLIP_CHUNK, a.n[t]);
    if (a.kind[t] == CLIP_F32) chunk_step<CLIP_F32, MOM>(a, t, from, to, s, lr, mu, wd);
    else if (a.kind[t] == CLIP_BF16) chunk_step<CLIP_BF16, MOM>(a, t, from, to, s, lr, mu, wd);
    else chunk_step<CLIP_F16, MOM>(a, t, from, to, s, lr, mu, wd);
  }
}

static unsigned clip_grid(long chunks) { return (unsigned)(chunks < CLIP_BLOCKS ? chunks : CLIP_BLOCKS); }

template <typename A>
static long fill_chunks(A& a, const long* n, const int* kind, int count) {
  long chunks = 0;
  a.count = count;
  for (int i = 0; i < count; ++i) {
    a.n[i] = n[i];
    a.kind[i] = (unsigned char)kind[i];
    a.first[i] = (int)chunks;
    chunks += (n[i] + CLIP_CHUNK - 1) / CLIP_CHUNK;
  }
  a.first[count] = (int)chunks;
  return chunks;
}

// blocks' sums that the norm of `count` tensors needs room for
extern "C" long lah_clip_partials(int count) {
  return (long)((count + CLIP_TENSORS - 1) / CLIP_TENSORS) * CLIP_BLOCKS;
}

extern "C" void lah_grad_norm(void* const* p, const long* n, const int* kind, int count, void* partial,
                              float max_norm, float eps, void* norm, void* scale, hipStream_t stream) {
  int used = 0;
  for (int i = 0; i < count; i += CLIP_TENSORS) {
    ClipTensors a;
    const int c = count - i < CLIP_TENSORS ? count - i : CLIP_TENSORS;
    const long chunks = fill_chunks(a, n + i, kind + i, c);
    for (int j = 0; j < c; ++j) a.p[j] = p[i + j];
    if (chunks == 0) continue;
    hipLaunchKernelGGL(clip_squares_kernel, dim3(clip_grid(chunks)), dim3(256), 0, stream, a,
                       (double*)partial + used);
    used += (int)clip_grid(chunks);
  }
  hipLaunchKernelGGL(clip_finish_kernel, dim3(1), dim3(1024), 0, stream, (const double*)partial, used,
                     max_norm, eps, (float*)norm, (float*)scale);
}

extern "C" void lah_grad_scale(void* const* p, const long* n, const int* kind, int count, const void* scale,
                               hipStream_t stream) {
  for (int i = 0; i < count; i += CLIP_TENSORS) {
    ClipTensors a;
    const int c = count - i < CLIP_TENSORS ? count - i : CLIP_TENSORS;
    const long chunks = fill_chunks(a, n + i, kind + i, c);
    for (int j = 0; j < c; ++j) a.p[j] = p[i + j];
    if (chunks > 0)
      hipLaunchKernelGGL(clip_scale_kernel, dim3(clip_grid(chunks)), dim3(256), 0, stream, a,
                         (const float*)scale);
  }
}

extern "C" void lah_master_sgd(void* const* p, void* const* m, void* const* g, void* const* b, const long* n,
                               const int* kind, int count, const void* scale, float lr, float mu, float wd,
                               hipStream_t stream) {
  for (int i = 0; i < count; i += CLIP_TENSORS) {
    StepTensors a;
    const int c = count - i < CLIP_TENSORS ? count - i : CLIP_TENSORS;
    const long chunks = fill_chunks(a, n + i, kind + i, c);
    for (int j = 0; j < c; ++j) {
      a.p[j] = (__bf16*)p[i + j];
      a.m[j] = (float*)m[i + j];
      a.g[j] = g[i + j];
      a.b[j] = b != nullptr ? (float*)b[i + j] : nullptr;
    }
    if (chunks == 0) continue;
    if (b != nullptr)
      hipLaunchKernelGGL((master_sgd_kernel<true>), dim3(clip_grid(chunks)), dim3(256), 0, stream, a,
                         (const float*)scale, lr, mu, wd);
    else
      hipLaunchKernelGGL((master_sgd_kernel<false>), dim3(clip_grid(chunks)), dim3(256), 0, stream, a,
                         (const float*)scale, lr, mu, wd);
  }
}
