// Matrix products grouped by expert with ragged sizes, for MI355X (gfx950).
//
//   forward   y[r]  = act(W[e] x[r] + b[e])          offsets[e] <= r < offsets[e+1]
//   dx        dx[r] = W[e]^T dP[r]
//   dW        dW[e] = sum_r dP[r] x[r]^T,  db[e] = sum_r dP[r]
//
// The rows of one expert stand together; how many each has is known on the GPU
// alone (offsets, [E+1] int32), so nothing here waits for the host and every
// launch can be captured. No row is padded: a row past an expert's end is
// loaded as zeros (the buffer descriptor's range check) and never stored.
//
// One tile kernel serves the three products. P is the operand whose index
// becomes the output's fast axis, Q the other one:
//             P                         Q                    contraction
//   NT fwd    W[e]  [N][K]   (KC)       x   rows  (KC)       K
//   NN dx     W[e]  [Kc][N]  (KS)       dP  rows  (KC)       Kc
//   TN dW     x     [r][N]   (KS)       dP  [r][M] (KS)      rows of e
// KC: the contraction is the operand's fast axis; a fragment is one 16-byte LDS
// read. KS: it is the slow axis; the fragment is read transposed from LDS
// (ds_read_b64_tr_b16), so no transposed copy of a weight is needed.
#include "common.h"

#define RBK 32  // contraction steps of a stage

enum { R_NT = 0, R_NN = 1, R_TN = 2 };
enum { R_PLAIN = 0, R_GELU = 1, R_GELU_DER = 2, R_MUL = 3 };  // forward epilogues
enum { R_F32 = 0, R_F32_ACC = 1, R_BF16 = 2 };                // dW outputs

typedef __attribute__((ext_vector_type(4))) int i32x4;
#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

LAH_DEVINL unsigned lds_addr(const void* p) {
  return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char*)p;
}

// Buffer descriptor of `bytes` from p: loads past them give zeros.
LAH_DEVINL i32x4 make_rsrc(const void* p, long bytes) {
  const unsigned long long a = (unsigned long long)p;
  const long b = bytes < 0 ? 0 : (bytes > 0x7fffffffL ? 0x7fffffffL : bytes);
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)((a >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane((int)b);
  r[3] = 0x00027000;
  return r;
}
#define OOB_OFFSET 0x80000000u  // past every descriptor made here

// Global -> LDS without registers, 16 bytes a lane, to lds + lane * 16. In asm,
// since the compiler would wait for every such load before the next LDS read;
// the stages' own counted waits order them here. It has no output register.
LAH_DEVINL void lds_load16(i32x4 rsrc, unsigned voff, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      ::"s"(lds), "v"(voff), "s"(rsrc)
      : "memory");
}

// All LDS reads of this wave done and at most N loads in flight, then the barrier.
template <int N>
LAH_DEVINL void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// LDS places of 16-byte chunks, so that the 16 lanes that read together hit 16
// different places mod 256 bytes (64 banks):
//  KC tile [rows][32]: 4 chunks a row; the chunk is XORed with two row bits. P's
//  rows come in steps of FN*4 (see p_row), so P takes its two bits there.
//  KS tile [32][cols]: a transposed read takes 2 chunks of each of 8 rows
//  {0..3, 8..11} (+4, +16); three row bits move the chunk pair.
template <int SHIFT>
LAH_DEVINL int kc_swz(int row) { return (row >> SHIFT) & 3; }
LAH_DEVINL int ks_swz(int row) { return ((row & 3) | ((row >> 1) & 4)) << 1; }

LAH_DEVINL float gelu_of(float x) {  // x * sigmoid(2u): one exp2, one reciprocal
  const float x2 = x * x;
  const float z = x * (-2.302208198f - 0.1029432397f * x2);  // -2u * log2(e)
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z));
}

LAH_DEVINL void gelu_and_slope(float x, float* g, float* d) {
  const float x2 = x * x;
  const float z = x * (-2.302208198f - 0.1029432397f * x2);
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z));
  const float du = 1.595769122f + 0.2140644488f * x2;  // 2u'
  *g = x * s;
  *d = s + x * (s - s * s) * du;
}

// The slot tables' search. M-tile slots of expert e start at s(e) = off[e]/BM + e:
// s(e+1) - s(e) = off[e+1]/BM - off[e]/BM + 1 covers its ceil(count/BM) tiles, and
// s grows with e, so the tile of a slot is found from the offsets alone, by
// counting the starts that are <= the slot, 64 a ballot. e == E: rows of nobody.
template <int BM>
LAH_DEVINL int find_expert(const int* __restrict__ offsets, int E, int slot) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b = 0; b <= E; b += 256) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = b + j * 64 + lane;
      const int o = e > 0 && e <= E ? offsets[e] : 0;
      n += __popcll(__ballot(e <= E && o / BM + e <= slot));
    }
  }
  return n - 1;
}

struct RaggedArgs {
  const __bf16* P;
  const __bf16* Q;
  void* C;
  const int* offsets;
  const void* bias;  // NT: [E, N]; fp32 or bf16
  __bf16* der;       // NT with slope: out; NN with R_MUL: in
  void* db;          // TN: [E, M] or null; fp32 or bf16
  long R;
  int E, N, M, K;    // K: contraction of NT / NN
  int bias_bf16;     // of bias, or of db
};

template <int KIND, int EPI, int WN, int WM, int FN, int FM, int STAGES>
__launch_bounds__(WN * WM * 64, 2) __global__ void ragged_gemm_kernel(RaggedArgs a) {
  constexpr int BN = WN * FN * 16, BM = WM * FM * 16, T = WN * WM * 64;
  constexpr bool P_KC = KIND == R_NT, Q_KC = KIND != R_TN;
  constexpr int PL = BN * RBK / 8 / T, QL = BM * RBK / 8 / T;  // loads a thread and stage
  constexpr int STAGE = (BN + BM) * RBK;                       // elements
  constexpr int PSHIFT = FN == 8 ? 5 : 4;                      // log2(FN * 4)
  static_assert(BN * RBK / 8 % T == 0 && BM * RBK / 8 % T == 0, "whole loads");
  static_assert(FN == 8 || FN == 4, "p_row and its swizzle");
  __shared__ __attribute__((aligned(16))) __bf16 smem[STAGES * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;

  // Blocks go to the 8 XCDs in turn: of each 512, the 64 that share one XCD
  // (two a CU) take 64 neighbouring tiles, whose operands then share its L2.
  int L = blockIdx.x;
  if (L < ((int)gridDim.x & ~511)) L = (L & ~511) | ((L & 7) << 6) | ((L >> 3) & 63);
  const int NT = cdiv(a.N, BN);

  int e, m0, n0, rows, steps;
  long row0;
  if (KIND == R_TN) {
    const int MT = cdiv(a.M, BM);
    e = L / (MT * NT);
    const int q = L % (MT * NT);
    const int first = q / (8 * NT) * 8, size = min(MT - first, 8), in = q % (8 * NT);
    m0 = (first + in % size) * BM;
    n0 = in / size * BN;
    const long lo = e == 0 ? 0 : min((long)max(a.offsets[e], 0), a.R);
    const long hi = min(max((long)a.offsets[e + 1], lo), a.R);
    row0 = lo;
    rows = (int)(hi - lo);
    steps = cdiv(rows, RBK);
  } else {
    e = find_expert<BM>(a.offsets, a.E, L / NT);
    e = __builtin_amdgcn_readfirstlane(e);
    const long lo = e == 0 ? 0 : min((long)max(a.offsets[e], 0), a.R);
    const long hi = e == a.E ? a.R : min(max((long)a.offsets[e + 1], lo), a.R);
    const int s0 = (int)(lo / BM) + e, slots = (int)(hi / BM) - (int)(lo / BM) + 1;
    // 8 M-tiles by all N-tiles at a time: neighbours share rows and weights
    const int q = L - s0 * NT;
    const int first = q / (8 * NT) * 8, size = min(slots - first, 8), in = q % (8 * NT);
    m0 = (first + in % size) * BM;
    n0 = in / size * BN;
    row0 = lo + m0;
    if (q < 0 || size <= 0 || row0 >= hi || n0 >= a.N) return;  // also where offsets do not ascend
    rows = (int)min(hi - row0, (long)BM);
    steps = e == a.E ? 0 : cdiv(a.K, RBK);
  }

  // ---- staging: each thread's byte offsets in its tile are the same in every step
  const __bf16 *Pb, *Qb;
  long pbytes, qbytes;  // from the base to the end of what may be read
  long pstep, qstep;    // elements from one stage to the next
  if (KIND == R_NT) {
    Pb = a.P + ((long)e * a.N + n0) * a.K;
    pbytes = (long)min(a.N - n0, BN) * a.K * 2;
    pstep = RBK;
  } else if (KIND == R_NN) {
    Pb = a.P + (long)e * a.K * a.N + n0;
    pbytes = ((long)a.K * a.N - n0) * 2;
    pstep = (long)RBK * a.N;
  } else {
    Pb = a.P + row0 * a.N + n0;
    pbytes = ((long)rows * a.N - n0) * 2;
    pstep = (long)RBK * a.N;
  }
  if (KIND == R_TN) {
    Qb = a.Q + row0 * a.M + m0;
    qbytes = ((long)rows * a.M - m0) * 2;
    qstep = (long)RBK * a.M;
  } else {
    Qb = a.Q + row0 * a.K;
    qbytes = (long)rows * a.K * 2;
    qstep = RBK;
  }
  unsigned pv[PL], qv[QL];
  int pc[PL], qc[QL];  // KC: the chunk's first contraction index
#pragma unroll
  for (int i = 0; i < PL; ++i) {
    const int idx = i * T + tid;
    if (P_KC) {
      const int r = idx >> 2, c = (idx & 3) ^ kc_swz<PSHIFT>(r);
      pv[i] = (unsigned)((long)r * a.K * 2 + c * 16);
      pc[i] = c * 8;
    } else {
      const int r = idx / (BN / 8), c = (idx % (BN / 8)) ^ ks_swz(r);
      pv[i] = (unsigned)((long)r * a.N * 2 + c * 16);
    }
  }
#pragma unroll
  for (int i = 0; i < QL; ++i) {
    const int idx = i * T + tid;
    if (Q_KC) {
      const int r = idx >> 2, c = (idx & 3) ^ kc_swz<2>(r);
      qv[i] = (unsigned)((long)r * a.K * 2 + c * 16);
      qc[i] = c * 8;
    } else {
      const int r = idx / (BM / 8), c = (idx % (BM / 8)) ^ ks_swz(r);
      qv[i] = (unsigned)((long)r * a.M * 2 + c * 16);
    }
  }
  const unsigned lds0 = lds_addr(smem) + wave * 1024;

  auto stage = [&](int t, int buf) {
    const unsigned to = lds0 + buf * STAGE * 2;
    const i32x4 rp = make_rsrc(Pb + t * pstep, pbytes - t * pstep * 2);
    const i32x4 rq = make_rsrc(Qb + t * qstep, qbytes - t * qstep * 2);
    // chunks past the contraction's end, which only a KC tile can hold, give zeros
    const int left = KIND == R_TN ? RBK : a.K - t * RBK;
#pragma unroll
    for (int i = 0; i < PL; ++i)
      lds_load16(rp, P_KC && pc[i] >= left ? OOB_OFFSET : pv[i], to + i * T * 16);
#pragma unroll
    for (int i = 0; i < QL; ++i)
      lds_load16(rq, Q_KC && qc[i] >= left ? OOB_OFFSET : qv[i], to + BN * RBK * 2 + i * T * 16);
  };

  f32x4 acc[FN][FM];
  f32x4 dbacc[KIND == R_TN ? FM : 1];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < (KIND == R_TN ? FM : 1); ++j) dbacc[j] = {0.f, 0.f, 0.f, 0.f};
  const bool with_db = KIND == R_TN && a.db != nullptr && n0 == 0 && wn == 0;
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.0f;

  // Fragment f, index i of P is tile row p_row: a lane's results in D rows
  // 4g..4g+3 of all FN fragments are then FN*4 neighbouring outputs (KC only).
  auto p_row = [&](int f) { return wn * FN * 16 + (l15 >> 2) * (FN * 4) + f * 4 + (l15 & 3); };

  auto read_ks = [&](const __bf16* tile, int cols, int base) {
    // lane i of 16 gets column base + i at 4 rows; lanes' addresses: row i >> 2, columns 4 (i & 3)
    const int r = g * 8 + (l15 >> 2), col = base + 4 * (l15 & 3);
    const int c0 = ((col >> 3) ^ ks_swz(r)) * 8 + (col & 7);
    const int c1 = ((col >> 3) ^ ks_swz(r + 4)) * 8 + (col & 7);
    bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, tile + r * cols + c0));
    bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, tile + (r + 4) * cols + c1));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  for (int t = 0; t < STAGES - 1 && t < steps; ++t) stage(t, t);
  int buf = 0;
  for (int t = 0; t < steps; ++t) {
    // stage t has landed; every wave is past its reads of stage t - 1, whose place is refilled
    if (t + STAGES - 2 < steps) wait_and_barrier<(STAGES - 2) * (PL + QL)>();
    else wait_and_barrier<0>();
    if (t + STAGES - 1 < steps) stage(t + STAGES - 1, buf == 0 ? STAGES - 1 : buf - 1);
    const __bf16* tp = smem + buf * STAGE;
    const __bf16* tq = tp + BN * RBK;
    bf16x8 pf[FN], qf[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      if (Q_KC) {
        const int r = wm * FM * 16 + j * 16 + l15;
        qf[j] = *(const bf16x8*)(tq + r * RBK + (g ^ kc_swz<2>(r)) * 8);
      } else {
        qf[j] = read_ks(tq, BM, wm * FM * 16 + j * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      if (P_KC) {
        const int r = p_row(i);
        pf[i] = *(const bf16x8*)(tp + r * RBK + (g ^ kc_swz<PSHIFT>(r)) * 8);
      } else {
        pf[i] = read_ks(tp, BN, wn * FN * 16 + i * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[i], qf[j], acc[i][j], 0, 0, 0);
    if (KIND == R_TN && with_db) {
#pragma unroll
      for (int j = 0; j < FM; ++j)
        dbacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, qf[j], dbacc[j], 0, 0, 0);
    }
    buf = buf == STAGES - 1 ? 0 : buf + 1;
  }

  // ---- epilogue: lane (l15, g) holds output row 16j + l15
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int r = wm * FM * 16 + j * 16 + l15;
    if (KIND == R_TN) {
      if (m0 + r < a.M) {
        const long at = ((long)e * a.M + m0 + r) * a.N;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const int n = n0 + wn * FN * 16 + i * 16 + g * 4;
          if (n < a.N) {
            if (EPI == R_BF16) {
              bf16x4 o;
#pragma unroll
              for (int q = 0; q < 4; ++q) o[q] = f2bf(acc[i][j][q]);
              *(bf16x4*)((__bf16*)a.C + at + n) = o;
            } else {
              float* c = (float*)a.C + at + n;
              *(f32x4*)c = EPI == R_F32_ACC ? *(const f32x4*)c + acc[i][j] : acc[i][j];
            }
          }
        }
        if (with_db && g == 0) {  // all 16 D rows hold the same sums
          const long at_b = (long)e * a.M + m0 + r;
          if (a.bias_bf16) ((__bf16*)a.db)[at_b] = f2bf(dbacc[j][0]);
          else ((float*)a.db)[at_b] = (EPI == R_F32_ACC ? ((float*)a.db)[at_b] : 0.f) + dbacc[j][0];
        }
      }
    } else if (r < rows) {
      const long at = (row0 + r) * a.N;
      constexpr int STEP = P_KC ? 8 : 4;  // neighbouring outputs stored at once
#pragma unroll
      for (int i0 = 0; i0 < FN; i0 += STEP / 4) {
        const int n = n0 + wn * FN * 16 + (P_KC ? g * (FN * 4) + i0 * 4 : i0 * 16 + g * 4);
        if (n < a.N) {
          float v[STEP];
#pragma unroll
          for (int q = 0; q < STEP; ++q) v[q] = acc[i0 + q / 4][j][q & 3];
          if (KIND == R_NT && a.bias != nullptr && e < a.E) {
            if (a.bias_bf16) {
              const bf16x8 b = *(const bf16x8*)((const __bf16*)a.bias + (long)e * a.N + n);
#pragma unroll
              for (int q = 0; q < STEP; ++q) v[q] += bf2f(b[q & 7]);
            } else {
#pragma unroll
              for (int h = 0; h < STEP; h += 4) {
                const f32x4 b = *(const f32x4*)((const float*)a.bias + (long)e * a.N + n + h);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[h + q] += b[q];
              }
            }
          }
          typedef __attribute__((ext_vector_type(STEP))) __bf16 outv;
          outv o, d;
          if (EPI == R_MUL) d = *(const outv*)(a.der + at + n);
#pragma unroll
          for (int q = 0; q < STEP; ++q) {
            if (EPI == R_GELU) {
              o[q] = f2bf(gelu_of(v[q]));
            } else if (EPI == R_GELU_DER) {
              float y, s;
              gelu_and_slope(v[q], &y, &s);
              o[q] = f2bf(y);
              d[q] = f2bf(s);  // the slope, in the outputs' type: one rounding of dP more
            } else if (EPI == R_MUL) {
              o[q] = f2bf(v[q] * bf2f(d[q]));
            } else {
              o[q] = f2bf(v[q]);
            }
          }
          *(outv*)((__bf16*)a.C + at + n) = o;
          if (EPI == R_GELU_DER) *(outv*)(a.der + at + n) = d;
        }
      }
    }
  }
}

template <int KIND, int EPI>
static void launch_ragged(const RaggedArgs& a, hipStream_t stream) {
  constexpr int WN = 2, WM = 2, FN = 8, FM = 4, BN = WN * FN * 16, BM = WM * FM * 16;
  const long nt = (a.N + BN - 1) / BN;
  const long tiles = KIND == R_TN ? (long)a.E * ((a.M + BM - 1) / BM) * nt
                                  : (a.R / BM + a.E + 1) * nt;
  hipLaunchKernelGGL((ragged_gemm_kernel<KIND, EPI, WN, WM, FN, FM, 3>), dim3((unsigned)tiles),
                     dim3(WN * WM * 64), 0, stream, a);
}

extern "C" void lah_ragged_nt(const void* x, const void* w, void* y, const void* offsets,
                              const void* bias, int bias_bf16, void* der, long R, int E, int N,
                              int K, int epi, hipStream_t stream) {
  RaggedArgs a{(const __bf16*)w, (const __bf16*)x, y, (const int*)offsets, bias, (__bf16*)der,
               nullptr, R, E, N, 0, K, bias_bf16};
  if (epi == R_GELU_DER) launch_ragged<R_NT, R_GELU_DER>(a, stream);
  else if (epi == R_GELU) launch_ragged<R_NT, R_GELU>(a, stream);
  else launch_ragged<R_NT, R_PLAIN>(a, stream);
}

// dx[r] = W[e]^T d[r] (times der[r], if given): W [E, K, N], d [R, K], out [R, N]
extern "C" void lah_ragged_nn(const void* d, const void* w, void* out, const void* offsets,
                              void* der, long R, int E, int N, int K, hipStream_t stream) {
  RaggedArgs a{(const __bf16*)w, (const __bf16*)d, out, (const int*)offsets, nullptr,
               (__bf16*)der, nullptr, R, E, N, 0, K, 0};
  if (der != nullptr) launch_ragged<R_NN, R_MUL>(a, stream);
  else launch_ragged<R_NN, R_PLAIN>(a, stream);
}

// dw[e] = sum_r d[r] x[r]^T: d [R, M], x [R, N], dw [E, M, N]; db [E, M] or null
extern "C" void lah_ragged_tn(const void* d, const void* x, void* dw, void* db, int db_bf16,
                              const void* offsets, long R, int E, int N, int M, int out,
                              hipStream_t stream) {
  RaggedArgs a{(const __bf16*)x, (const __bf16*)d, dw, (const int*)offsets, nullptr, nullptr,
               db, R, E, N, M, 0, db_bf16};
  if (out == R_BF16) launch_ragged<R_TN, R_BF16>(a, stream);
  else if (out == R_F32_ACC) launch_ragged<R_TN, R_F32_ACC>(a, stream);
  else launch_ragged<R_TN, R_F32>(a, stream);
}
