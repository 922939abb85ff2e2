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
// P is the operand whose index becomes the output's fast axis, Q the other one:
//             P                         Q                    contraction
//   NT fwd    W[e]  [N][K]   (KC)       x   rows  (KC)       K
//   NN dx     W[e]  [Kc][N]  (KS)       dP  rows  (KC)       Kc
//   TN dW     x     [r][N]   (KS)       dP  [r][M] (KS)      rows of e
// KC: the contraction is the operand's fast axis; a fragment is one 16-byte LDS
// read. KS: it is the slow axis; the fragment is read transposed from LDS
// (ds_read_b64_tr_b16), so no transposed copy of a weight is needed.
//
// Three kernels: 256 x 256 tiles by one persistent block a CU (ragged_big_kernel: all dW,
// and rows where experts have many), 128 x 256 tiles by two blocks a CU (ragged_rows_kernel)
// and 16 x 16 tiles that read weights past LDS (ragged_few_kernel: decoded tokens). The
// first is bound by the matrix cores with their power limit, the others by reading weights.
#include "common.h"
#include <type_traits>
#include <utility>

#define RBK 32   // contraction steps of a phase of KS operands
#define RBN 256  // P's side of a tile
#define RBM 128  // Q's side
#define RT 256   // threads

enum { R_NT = 0, R_NN = 1, R_TN = 2 };
enum { R_PLAIN = 0, R_GELU = 1, R_GELU_DER = 2, R_MUL = 3, R_PART = 4 };  // epilogues of rows; fp32 sums of a part
enum { R_F32 = 0, R_F32_ACC = 1, R_BF16 = 2 };                // dW outputs

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
#define LDS_PTR(T, p) ((__attribute__((address_space(3))) T*)(p))

LAH_DEVINL unsigned lds_addr(const void* p) {
  return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char*)p;
}

// Buffer descriptor of `bytes` from p: loads past them give zeros.
LAH_DEVINL i32x4 make_rsrc(const void* p, int bytes) {
  const unsigned long long a = (unsigned long long)p;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)((a >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane(bytes);
  r[3] = 0x00027000;
  return r;
}
// A load in asm may not read a scalar register that a vector instruction (such as the
// readfirstlane above) wrote less than five instructions ago, and the compiler does not look
// into it: the descriptor is held in scalar registers from here on, and five stand between.
LAH_DEVINL i32x4 settled_rsrc(const void* p, int bytes) {
  i32x4 r = make_rsrc(p, bytes);
  asm volatile("s_nop 4" : "+s"(r));
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

// the same, of what need not stay in L2
LAH_DEVINL void lds_load16_once(i32x4 rsrc, unsigned voff, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen nt lds"
      ::"s"(lds), "v"(voff), "s"(rsrc)
      : "memory");
}

// All LDS reads of this wave done and at most N loads in flight, then the barrier.
template <int N>
LAH_DEVINL void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int N>
LAH_DEVINL void wait_loads_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

LAH_DEVINL void wait_reads_and_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// LDS places of 16-byte chunks, so that the 16 lanes that are served together hit
// 16 different places mod 256 bytes (64 banks).
//  KC tile [rows][64], 8 chunks a row: a 16-byte read serves quads of lanes q = 0, 3
//  of one 16 and 1, 2 of the next together, and the others. Chunks are XORed with
//  0 2 3 1 by the quad's row bits, and the row's second bit on top (counted: no
//  conflict; the quad's bits themselves conflict two ways).
//  KS tile [32][cols]: a transposed read takes 2 chunks of each of 8 rows
//  {0..3, 8..11} (+4, +16); three row bits move the chunk pair.
template <int SHIFT>
LAH_DEVINL int kc_swz(int row) {
  const int q = (row >> SHIFT) & 3;
  return ((row & 2) << 1) | (((q << 1) ^ q) & 2) | (q >> 1);
}
LAH_DEVINL int ks_swz(int row) { return ((row & 3) | ((row >> 1) & 4)) << 1; }

// Fragment of a KS tile: lane i of 16 gets column base + i at rows 8g .. 8g + 7.
LAH_DEVINL bf16x8 read_ks(const __bf16* tile, int cols, int base, int lane) {
  const int l15 = lane & 15, r = (lane >> 4) * 8 + (l15 >> 2), col = base + 4 * (l15 & 3);
  const int c0 = ((col >> 3) ^ ks_swz(r)) * 8 + (col & 7);
  const int c1 = ((col >> 3) ^ ks_swz(r + 4)) * 8 + (col & 7);
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, tile + r * cols + c0));
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(LDS_PTR(bf16x4, tile + (r + 4) * cols + c1));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

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
  _Float16* der;     // gelu's slope, below 1.13: 11 bits where bf16 has 8. NT: out; NN with R_MUL: in
  void* db;          // TN: [E, M] or null; fp32 or bf16
  long R;
  int E, N, M, K;    // K: contraction of NT / NN
  int bias_bf16;     // of bias, or of db
  int splits;        // parts of the contraction, each with sums of its own
  bool once;         // weights that no cache holds until they are read again
};

// Blocks go to the 8 XCDs in turn: of each 512, the 64 that share one XCD (two a
// CU) take 64 neighbouring tiles, whose operands then share its L2.
LAH_DEVINL int xcd_tile() {
  const int L = blockIdx.x;
  return L < ((int)gridDim.x & ~511) ? (L & ~511) | ((L & 7) << 6) | ((L >> 3) & 63) : L;
}

// rows [lo, hi) of expert e, whatever the offsets hold
LAH_DEVINL void expert_rows(const RaggedArgs& a, int e, long* lo, long* hi) {
  *lo = e == 0 ? 0 : min((long)max(a.offsets[e], 0), a.R);
  *hi = e == a.E ? a.R : min(max((long)a.offsets[e + 1], *lo), a.R);
}

#define MFMA(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0)

// ---------------------------------------------------------------------------
// forward (NT) and dx (NN): rows of Q against one expert's weight
//
// A block is 4 waves on a tile of 128 Q by 256 P, a wave 64 by 128: 128 accumulators a
// lane, so that two blocks share a CU and one's epilogue hides under the other's products.
// 1024 experts of 32 rows, 2048 -> 512: 431 us, 2.3 GB at 5.4 TB/s, its dx 453.
//
// A stage is 64 contraction steps, so that KC rows are whole 128-byte lines (at 32
// the same loads are twice the requests: 740 against 1000 TFLOP/s). It runs in two
// phases of 32 MFMAs a wave: NT takes half of P's rows in each (Q's fragments stay
// in registers), NN half of the contraction. P rides in a ring of 3 half stages, Q
// in 2 whole ones: 80 KB, just two blocks a CU, and every load has two phases to land.
// ---------------------------------------------------------------------------
template <int KIND, int EPI>
__launch_bounds__(RT, 2) __global__ void ragged_rows_kernel(RaggedArgs a) {
  constexpr bool P_KC = KIND == R_NT;
  constexpr int SLOT = 8192;  // elements: 128 x 64 (KC) or 32 x 256 (KS)
  __shared__ __attribute__((aligned(16))) __bf16 smem[5 * SLOT];

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = wave >> 1;

  const int L = xcd_tile(), NT = cdiv(a.N, RBN);
  const int e = __builtin_amdgcn_readfirstlane(find_expert<RBM>(a.offsets, a.E, L / NT));
  long lo, hi;
  expert_rows(a, e, &lo, &hi);
  const int s0 = (int)(lo / RBM) + e, slots = (int)(hi / RBM) - (int)(lo / RBM) + 1;
  // 8 M-tiles by all N-tiles at a time: neighbours share rows and weights
  const int q = L - s0 * NT;
  const int first = q / (8 * NT) * 8, size = min(slots - first, 8), in = q % (8 * NT);
  const int m0 = (first + in % size) * RBM, n0 = in / size * RBN;
  const long row0 = lo + m0;
  if (q < 0 || size <= 0 || row0 >= hi || n0 >= a.N) return;  // also where offsets do not ascend
  const int rows = (int)min(hi - row0, (long)RBM);
  const int all = e == a.E ? 0 : cdiv(a.K, 64);
  const int begin = EPI == R_PART ? all * (int)blockIdx.y / a.splits : 0;
  const int steps = EPI == R_PART ? all * ((int)blockIdx.y + 1) / a.splits : all;  // the end

  // ---- staging: a thread's byte offsets in a tile are the same in every stage
  const __bf16* Pb = a.P + ((long)e * a.N * a.K + (P_KC ? (long)n0 * a.K : n0));
  const __bf16* Qb = a.Q + row0 * a.K;
  // bytes from the base to the end of what may be read (below 2^31: N * K < 2^30, K < 2^21)
  const int pbytes = P_KC ? min(a.N - n0, RBN) * a.K * 2 : 0, qbytes = rows * a.K * 2;
  unsigned pv[4], qv[4];
  int cc[4];  // KC: a chunk's first contraction index
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int idx = i * RT + tid;
    const int r = idx >> 3, c = (idx & 7) ^ kc_swz<2>(r);
    qv[i] = (unsigned)(r * a.K + c * 8) * 2;
    cc[i] = c * 8;
    if (P_KC) {  // half h has rows 128 wn + 32 q + 16 h + ..: 16 of every 32
      const int pc = (idx & 7) ^ kc_swz<4>(r);
      pv[i] = (unsigned)(((r >> 4) * 32 + (r & 15)) * a.K + pc * 8) * 2;
    } else {
      const int kr = idx >> 5, pc = (idx & 31) ^ ks_swz(kr);
      pv[i] = (unsigned)(kr * a.N + pc * 8) * 2;
    }
  }
  int pcc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) pcc[i] = ((i * RT + tid) & 7 ^ kc_swz<4>((i * RT + tid) >> 3)) * 8;
  const unsigned lds0 = lds_addr(smem) + wave * 1024;

  auto load4 = [&](const i32x4& r, auto at, unsigned to) {
    if (a.once) {
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_load16_once(r, at(i), to + i * RT * 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) lds_load16(r, at(i), to + i * RT * 16);
    }
  };
  auto stage_p = [&](int p) {  // phase p's part, to slot p % 3
    const int t = p >> 1, h = p & 1;
    const unsigned to = lds0 + (p % 3) * (SLOT * 2);
    if (P_KC) {
      const int skip = h * 16 * a.K + t * 64;
      const i32x4 r = settled_rsrc(Pb + skip, max(pbytes - skip * 2, 0));  // few columns: no second half
      const int left = a.K - t * 64;
      load4(r, [&](int i) { return pcc[i] >= left ? OOB_OFFSET : pv[i]; }, to);
    } else {
      const int left = max(min(a.K - p * RBK, RBK), 0);
      const i32x4 r = settled_rsrc(Pb + (long)p * RBK * a.N, left > 0 ? (left * a.N - n0) * 2 : 0);
      load4(r, [&](int i) { return pv[i]; }, to);
    }
  };
  auto stage_q = [&](int t) {
    const unsigned to = lds0 + (3 + (t & 1)) * (SLOT * 2);
    const i32x4 r = settled_rsrc(Qb + t * 64, qbytes - t * 128);
    const int left = a.K - t * 64;  // chunks past the contraction's end give zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) lds_load16(r, cc[i] >= left ? OOB_OFFSET : qv[i], to + i * RT * 16);
  };

  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = {0.f, 0.f, 0.f, 0.f};

  // P's fragment i, lane l15 is tile row 128 wn + 32 (l15 / 4) + 4 i + l15 % 4: a
  // lane's results in D rows 4g .. 4g+3 of all 8 are then 32 neighbouring outputs.
  const int prow = wn * 64 + (l15 >> 2) * 16 + (l15 & 3);  // in a half's slot, + 4 (i & 3)
  const int qrow = wm * 64 + l15;
  auto read_q = [&](int t, int j, int kk) {
    const int r = qrow + j * 16;
    return *(const bf16x8*)(smem + (3 + (t & 1)) * SLOT + r * 64 + ((kk * 4 + g) ^ kc_swz<2>(r)) * 8);
  };
  auto read_p_kc = [&](int p, int i, int kk) {
    const int r = prow + i * 4;
    return *(const bf16x8*)(smem + (p % 3) * SLOT + r * 64 + ((kk * 4 + g) ^ kc_swz<4>(r)) * 8);
  };

  if (begin < steps) {
    stage_p(2 * begin);
    stage_q(begin);
    stage_p(2 * begin + 1);
  }
  for (int t = begin; t < steps; ++t) {
    const bool more = t + 1 < steps;
    bf16x8 qf[4][2];
    // the phase's loads have landed; all waves are past their reads of what is refilled now
    wait_and_barrier<4>();
    if (more) {
      stage_p(2 * t + 2);
      stage_q(t + 1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qf[j][0] = read_q(t, j, 0);
      if (P_KC) qf[j][1] = read_q(t, j, 1);
    }
    bf16x8 pf[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      pf[i] = P_KC ? read_p_kc(2 * t, i & 3, i >> 2)
                   : read_ks(smem + (2 * t) % 3 * SLOT, RBN, wn * 128 + i * 16, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (P_KC) acc[i & 3][j] = MFMA(pf[i], qf[j][i >> 2], acc[i & 3][j]);
        else acc[i][j] = MFMA(pf[i], qf[j][0], acc[i][j]);
      }
    if (more) {
      wait_and_barrier<8>();
      stage_p(2 * t + 3);
    } else {
      wait_and_barrier<0>();
    }
    if (!P_KC) {
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[j][1] = read_q(t, j, 1);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      pf[i] = P_KC ? read_p_kc(2 * t + 1, i & 3, i >> 2)
                   : read_ks(smem + (2 * t + 1) % 3 * SLOT, RBN, wn * 128 + i * 16, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (P_KC) acc[4 + (i & 3)][j] = MFMA(pf[i], qf[j][i >> 2], acc[4 + (i & 3)][j]);
        else acc[i][j] = MFMA(pf[i], qf[j][1], acc[i][j]);
      }
  }

  // ---- epilogue: lane (l15, g) holds output row 16 j + l15
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = wm * 64 + j * 16 + l15;
    if (r >= rows) continue;
    const long at = (row0 + r) * a.N;
    constexpr int STEP = P_KC ? 8 : 4;  // neighbouring outputs stored at once
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += STEP / 4) {
      const int n = n0 + wn * 128 + (P_KC ? g * 32 + i0 * 4 : i0 * 16 + g * 4);
      if (n >= a.N) continue;
      float v[STEP];
#pragma unroll
      for (int x = 0; x < STEP; ++x) v[x] = acc[i0 + x / 4][j][x & 3];
      if (EPI == R_PART) {
        float* to = (float*)a.C + ((long)blockIdx.y * a.R * a.N + at + n);
#pragma unroll
        for (int h = 0; h < STEP; h += 4) *(f32x4*)(to + h) = f32x4{v[h], v[h + 1], v[h + 2], v[h + 3]};
        continue;
      }
      if (KIND == R_NT && a.bias != nullptr && e < a.E) {
        if (a.bias_bf16) {
          const bf16x8 b = *(const bf16x8*)((const __bf16*)a.bias + (long)e * a.N + n);
#pragma unroll
          for (int x = 0; x < STEP; ++x) v[x] += bf2f(b[x & 7]);
        } else {
#pragma unroll
          for (int h = 0; h < STEP; h += 4) {
            const f32x4 b = *(const f32x4*)((const float*)a.bias + (long)e * a.N + n + h);
#pragma unroll
            for (int x = 0; x < 4; ++x) v[h + x] += b[x];
          }
        }
      }
      typedef __attribute__((ext_vector_type(STEP))) __bf16 outv;
      typedef __attribute__((ext_vector_type(STEP))) _Float16 slopev;
      outv o;
      slopev d;
      if (EPI == R_MUL) d = *(const slopev*)(a.der + at + n);
#pragma unroll
      for (int x = 0; x < STEP; ++x) {
        if (EPI == R_GELU) {
          o[x] = f2bf(gelu_of(v[x]));
        } else if (EPI == R_GELU_DER) {
          float y, s;
          gelu_and_slope(v[x], &y, &s);
          o[x] = f2bf(y);
          d[x] = (_Float16)s;
        } else if (EPI == R_MUL) {
          o[x] = f2bf(v[x] * (float)d[x]);
        } else {
          o[x] = f2bf(v[x]);
        }
      }
      *(outv*)((__bf16*)a.C + at + n) = o;
      if (EPI == R_GELU_DER) *(slopev*)(a.der + at + n) = d;
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows (single decoded tokens, small products): an active expert's weight through the CUs
//
// Bound by HBM, or by latency. A block has 16 outputs of one expert for up to 16 of its
// rows, its 4 waves a quarter of the contraction each; the weight goes from global memory
// straight into the matrix instruction's registers, and the four sums meet in LDS. Blocks
// are counted by non-empty tiles, of which there are at most min(R, R / 16 + E + 1): a
// grid over all experts' slots would start 4112 blocks to find the 64 that one token
// needs (34 us, 1024 -> 4096 of 256 experts).
// ---------------------------------------------------------------------------
#define FR 16  // rows and outputs of a tile

// The tile'th of the tiles of 16 rows of all groups in order (group E: rows of nobody);
// -1 past the last. Each lane counts some neighbouring groups.
LAH_DEVINL int find_tile(const RaggedArgs& a, int tile, long* row0, int* rows) {
  const int lane = threadIdx.x & 63, per = (a.E + 64) / 64;
  int mine = 0;
#pragma unroll 4
  for (int j = 0; j < per; ++j) {
    const int e = lane * per + j;
    if (e <= a.E) {
      long lo, hi;
      expert_rows(a, e, &lo, &hi);
      mine += (int)((hi - lo + FR - 1) / FR);
    }
  }
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(upto, d, 64);
    if (lane >= d) upto += v;
  }
  // the lane whose groups hold the tile looks through them again
  int skip = tile - (upto - mine), found = -1, first = 0, count = 0;
#pragma unroll 4
  for (int j = 0; j < per; ++j) {
    const int e = lane * per + j;
    if (e <= a.E) {
      long lo, hi;
      expert_rows(a, e, &lo, &hi);
      const int n = (int)((hi - lo + FR - 1) / FR);
      if (skip >= 0 && skip < n) {
        found = e;
        first = (int)(lo + (long)skip * FR);
        count = (int)min(hi - lo - (long)skip * FR, (long)FR);
      }
      skip -= n;
    }
  }
  const unsigned long long has = __ballot(found >= 0);
  if (has == 0) return -1;
  const int owner = __builtin_amdgcn_readfirstlane(__ffsll(has) - 1);
  *row0 = __builtin_amdgcn_readlane(first, owner);
  *rows = __builtin_amdgcn_readlane(count, owner);
  return __builtin_amdgcn_readlane(found, owner);
}

template <int EPI>
__launch_bounds__(256) __global__ void ragged_few_kernel(RaggedArgs a, int per) {
  __shared__ __attribute__((aligned(16))) float part[2][4][16][20];  // [wave][row][output]; 20: rows 20 banks apart
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  long row0 = 0;
  int rows = 0;
  const int e = find_tile(a, blockIdx.y, &row0, &rows);
  if (e < 0) return;
  const bool nobody = e == a.E;
  const int chunks = cdiv(a.K, 32), c0 = chunks * wave / 4, c1 = chunks * (wave + 1) / 4;
  const bool row_ok = l15 < rows;
  const __bf16* x = a.Q + (row0 + (row_ok ? l15 : 0)) * a.K + g * 8;
  for (int n0 = blockIdx.x * per * FR, i = 0; i < per && n0 < a.N; ++i, n0 += FR) {
    f32x4 acc[2];
    acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!nobody) {
      const __bf16* w = a.P + ((long)e * a.N + min(n0 + l15, a.N - 1)) * a.K + g * 8;
      int c = c0;
      for (; c + 8 <= c1 && (c + 8) * 32 <= a.K; c += 8) {
        bf16x8 wf[8], xf[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) wf[u] = *(const bf16x8*)(w + (c + u) * 32);
#pragma unroll
        for (int u = 0; u < 8; ++u) xf[u] = row_ok ? *(const bf16x8*)(x + (c + u) * 32) : bf16x8{};
#pragma unroll
        for (int u = 0; u < 8; ++u) acc[u & 1] = MFMA(wf[u], xf[u], acc[u & 1]);
      }
      for (; c < c1; ++c) {
        const bool in = c * 32 + g * 8 < a.K;  // past the contraction's end: zeros
        const bf16x8 wf = in ? *(const bf16x8*)(w + c * 32) : bf16x8{};
        const bf16x8 xf = in && row_ok ? *(const bf16x8*)(x + c * 32) : bf16x8{};
        acc[0] = MFMA(wf, xf, acc[0]);
      }
    }
    float(*sums)[16][20] = part[i & 1];  // the other one is still read
    *(f32x4*)&sums[wave][l15][g * 4] = acc[0] + acc[1];
    __syncthreads();
    const int r = tid >> 4, n = n0 + (tid & 15);  // one output a thread
    if (r >= rows || n >= a.N) continue;
    float v = (sums[0][r][tid & 15] + sums[1][r][tid & 15]) + (sums[2][r][tid & 15] + sums[3][r][tid & 15]);
    if (a.bias != nullptr && !nobody) {
      const long at = (long)e * a.N + n;
      v += a.bias_bf16 ? bf2f(((const __bf16*)a.bias)[at]) : ((const float*)a.bias)[at];
    }
    const long at = (row0 + r) * a.N + n;
    if (EPI == R_GELU_DER) {
      float y, s;
      gelu_and_slope(v, &y, &s);
      ((__bf16*)a.C)[at] = f2bf(y);
      a.der[at] = (_Float16)s;
    } else {
      ((__bf16*)a.C)[at] = f2bf(EPI == R_GELU ? gelu_of(v) : v);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: 256 x 256 tiles, one persistent block of 4 waves a CU
//
// A wave has 128 x 128 of the tile, 256 accumulators a lane, and its SIMD to itself.
// Against 8 waves of 64 x 128 that is a third fewer LDS reads and half the scalar
// work a product, and what bounds large products on this card is power: at 4 x 8192
// rows, K = N = 4096, 8 waves ran 52 % of the MFMA cycles at 2.05 GHz.
//
// A CU has room for one such tile, so nothing else could hide its first loads and
// last stores: the block runs through a list of tiles and loads two stages ahead,
// into the next tile where the present one ends; stores are left in flight. A stage
// is 64 contraction steps of P and Q (32 KB each, two stages in LDS) in quarters of
// 32 MFMAs: two for each half of the steps. Each quarter reads 8 fragments of the
// next but one. P's place is free behind the first quarter and Q's behind the second
// (barriers, where no read is out) and both are loaded again; P of the next stage has
// landed before the third quarter, Q before the last: loads have a stage and a half
// (at a stage, the misses of L2 were waited for: 10 % more time).
//
// 256 experts, 262144 rows of uneven sizes, 1024 -> 4096, 2.2 TFLOP: forward 1997 us (1100
// TFLOP/s), with gelu 2239, dx 1950, dW 2167. Of an earlier forward's 2116 the stores were
// 330, the loads 420 and the LDS reads 180; 1150 is what its MFMAs take alone. Zeros in
// place of numbers take 1770: the rest is power.
// ---------------------------------------------------------------------------
#define BT 256
#define BM 256
#define BN 256
#define BSLOT 16384  // elements of one operand's stage

// M-tiles of all experts in order: table[0] = their number, then {expert, first
// row, rows, 0}. Rows of nobody come last, as expert E.
__launch_bounds__(1024) __global__ void ragged_tiles_kernel(const int* __restrict__ offsets, int E, long R,
                                                            int4* __restrict__ table) {
  __shared__ int start[4098];
  __shared__ int wsum[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PER = 5;  // E + 1 <= 4097 groups
  int c[PER], sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = tid * PER + j;
    c[j] = 0;
    if (e <= E) {
      const long lo = e == 0 ? 0 : min((long)max(offsets[e], 0), R);
      const long hi = e == E ? R : min(max((long)offsets[e + 1], lo), R);
      c[j] = (int)((hi - lo + BM - 1) / BM);
    }
    sum += c[j];
  }
  int inc = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(inc, d, 64);
    if (lane >= d) inc += v;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int at = inc - sum, total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    at += w < wave ? wsum[w] : 0;
    total += wsum[w];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (tid * PER + j <= E) start[tid * PER + j] = at;
    at += c[j];
  }
  // where offsets do not ascend, groups overlap: no more tiles than the table has room for
  const int most = (int)min((long)total, R / BM + E + 1);
  if (tid == 0) table[0] = make_int4(most, 0, 0, 0);
  __syncthreads();
  for (int i = tid; i < most; i += 1024) {
    int lo_e = 0, hi_e = E;  // the last group that starts at or before tile i has it
    while (lo_e < hi_e) {
      const int mid = (lo_e + hi_e + 1) >> 1;
      if (start[mid] <= i) lo_e = mid;
      else hi_e = mid - 1;
    }
    const int e = lo_e;
    const long lo = e == 0 ? 0 : min((long)max(offsets[e], 0), R);
    const long hi = e == E ? R : min(max((long)offsets[e + 1], lo), R);
    const long row0 = lo + (long)(i - start[e]) * BM;
    table[1 + i] = make_int4(e, (int)row0, (int)max(min(hi - row0, (long)BM), 0l), 0);
  }
}

// The accumulators of a wave that has its SIMD to itself fill the accumulation
// registers; the compiler's own products move them about (four copies before each, with
// the branches below). In asm it cannot see how long their results take: whatever else
// touches them stands behind settle(), 32 cycles.
LAH_DEVINL void mfma_acc(f32x4& c, const bf16x8& a, const bf16x8& b) {
  asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// a few more, in the other registers
LAH_DEVINL void mfma_vgpr(f32x4& c, const bf16x8& a, const bf16x8& b) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
LAH_DEVINL void settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
// the value is in its accumulation registers here, and read or written beyond
LAH_DEVINL void pin_acc(f32x4& c) { asm volatile("" : "+a"(c)); }

LAH_DEVINL void pin_vgpr(f32x4& c) { asm volatile("" : "+v"(c)); }

// lds_load16 in two parts, to a place at a fixed distance: where, and one instruction
// later (a matrix product, or s_nop) the load.
template <int AT>
LAH_DEVINL void lds_load_to(unsigned lds) {
  asm volatile("s_add_u32 m0, %0, %1" ::"s"(lds), "n"(AT) : "memory", "scc");
}
LAH_DEVINL void lds_load_go(i32x4 rsrc, unsigned voff) {
  asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc) : "memory");
}
LAH_DEVINL bf16x8 lds_read16(unsigned at, int off) {
  return *(__attribute__((address_space(3))) const bf16x8*)(at + off);
}
LAH_DEVINL bf16x8 lds_read_tr(unsigned at, int off, int four_rows) {
  typedef __attribute__((address_space(3))) bf16x4* place;
  const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((place)(at + off));
  const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((place)(at + off + four_rows));
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <typename F, int... X>
LAH_DEVINL void each_of(F&& f, std::integer_sequence<int, X...>) {
  (f(std::integral_constant<int, X>()), ...);
}
template <int N, typename F>
LAH_DEVINL void each(F&& f) { each_of(f, std::make_integer_sequence<int, N>()); }
template <int N>
using number = std::integral_constant<int, N>;

#define OUT_ROW 272  // bytes

// Stores of whole lines need not stay in L2, parts of lines meet there: dW of 1024 experts of
// 32 rows, 2048 x 512, 382 us and 517 where they stay, of 300 of 32 rows, 2936 x 1400, 886 and 655.
template <typename T, typename Rsrc>
LAH_DEVINL void store4(const T (&v)[4], Rsrc to, const unsigned (&off)[4], bool lines) {
  if (lines) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[k]), to, off[k], 0, 2);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v[k]), to, off[k], 0, 0);
  }
}

struct BigTile {
  int e, out = 0, rows, steps, m0, n0, q;  // out: dW's place
  long row0;
};

template <int KIND, int EPI>
__launch_bounds__(BT, 1) __global__ void ragged_big_kernel(RaggedArgs a, const int4* __restrict__ table) {
  constexpr bool P_KC = KIND == R_NT, Q_KC = KIND != R_TN;
  __shared__ __attribute__((aligned(16))) __bf16 smem[4 * BSLOT];
  __shared__ __attribute__((aligned(16))) float bias_lds[P_KC ? 4 : 1][BN];
  __shared__ __attribute__((aligned(16))) char turn_lds[P_KC ? 1 : 4][16 * OUT_ROW];  // a wave's 16 rows of 256 bytes

  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = wave >> 1;

  const int NT = cdiv(a.N, BN);
  // M-tiles of one expert, or of all
  const int MT = KIND == R_TN ? cdiv(a.M, BM) : __builtin_amdgcn_readfirstlane(table[0].x);
  const int groups = KIND != R_TN ? 1 : table == nullptr ? a.splits * a.E : __builtin_amdgcn_readfirstlane(table[0].x);
  const int tiles = groups * MT * NT;
  // 32 neighbouring tiles at a time on the 32 CUs of an XCD (blocks go to XCDs in turn)
  const int stride = gridDim.x;
  const int mine = stride % 256 == 0 ? (blockIdx.x & ~255) | ((blockIdx.x & 7) << 5) | ((blockIdx.x >> 3) & 31)
                                     : (int)blockIdx.x;

  // 4 M-tiles by all N-tiles at a time, so that an XCD has 4 by 8: 12 operand tiles for 32
  // products, where 8 by 4 of experts of 4 M-tiles has 16 (256 experts of 1024 rows, 1024 ->
  // 4096: 2022 us by 4, 2070 by 8, 2103 by 16; one expert 1891, 1967, 1957).
  auto decode = [&](int L) {
    BigTile w;
    int q = L;
    if (KIND == R_TN) {
      w.e = L / (MT * NT);
      q = L % (MT * NT);
    }
    const int first = q / (4 * NT) * 4, size = min(MT - first, 4), in = q % (4 * NT);
    const int m = first + in % size;
    w.q = q;
    w.n0 = in / size * BN;
    if (KIND == R_TN) {
      if (table != nullptr) {
        const int4 t = table[1 + w.e];
        w.e = t.x;
        w.row0 = t.y;
        w.rows = t.z;
        w.out = t.w;
      } else {  // parts of equal rows
        w.out = w.e;
        const int part = w.e / a.E;
        w.e -= part * a.E;
        long lo, hi;
        expert_rows(a, w.e, &lo, &hi);
        const long each = a.splits == 1 ? hi - lo : (((hi - lo) / a.splits + 64) & ~63L);
        w.row0 = min(lo + part * each, hi);
        w.rows = (int)min(each, hi - w.row0);
      }
      w.m0 = m * BM;
      w.steps = max(cdiv(w.rows, 64), 1);
    } else {
      const int4 t = table[1 + m];
      w.e = t.x;
      w.row0 = t.y;
      w.rows = t.z;
      w.m0 = 0;
      w.steps = w.e == a.E ? 1 : cdiv(a.K, 64);
    }
    w.e = __builtin_amdgcn_readfirstlane(w.e);
    w.rows = __builtin_amdgcn_readfirstlane(w.rows);
    w.steps = __builtin_amdgcn_readfirstlane(w.steps);
    w.q = __builtin_amdgcn_readfirstlane(w.q);
    w.out = __builtin_amdgcn_readfirstlane(w.out);
    w.row0 = (long)(unsigned)__builtin_amdgcn_readfirstlane((int)w.row0);
    return w;
  };

  // ---- staging: a thread's byte offsets are the same in every stage
  unsigned pv0[8], qv0[8];
  const int pr = P_KC ? tid >> 3 : tid >> 5, qr = Q_KC ? tid >> 3 : tid >> 4;
  const int pc = P_KC ? ((tid & 7) ^ kc_swz<3>(pr)) * 8 : 0;
  const int qc = Q_KC ? ((tid & 7) ^ kc_swz<2>(qr)) * 8 : ((tid & 15) ^ ks_swz(qr)) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // KC: row 128 w + 8 l + f of P, fragment f's lane l, is row 128 w + 32 (f / 2) + 8 (l / 4) +
    // 4 (f % 2) + l % 4 in LDS, where the reads have no conflicts
    const int lr = pr + i * 32, pf = (lr >> 5 & 3) * 2 + (lr >> 2 & 1), pl = (lr >> 3 & 3) * 4 + (lr & 3);
    pv0[i] = P_KC ? (unsigned)(((lr & 128) + pl * 8 + pf) * a.K + pc) * 2
                 : (unsigned)((pr + i * 8) * a.N + ((tid & 31) ^ ks_swz(pr + i * 8)) * 8) * 2;
    // KS: two tiles [64][128] beside each other
    qv0[i] = Q_KC ? (unsigned)((qr + i * 32) * a.K + qc) * 2
                 : (unsigned)((qr + (i & 3) * 16) * a.M + (i >> 2) * 128 + qc) * 2;
  }
  const unsigned lds0 = lds_addr(smem) + wave * 1024;
  const unsigned bias0 = lds_addr(bias_lds);

  // The stage that is loaded next: descriptors, contraction steps left, place. Within a
  // tile they move on by a few scalar additions.
  const char *pat = nullptr, *qat = nullptr;
  int pbytes = 0, qbytes = 0, left = 0;
  unsigned to = lds0;
  const long pstep = P_KC ? 128 : 128L * a.N, qstep = Q_KC ? 128 : 128L * a.M;  // bytes
  unsigned pv[8], qv[8];  // offsets in use: past everything where the contraction has ended
  auto mask_offsets = [&]() {  // KC: chunks past the contraction's end give zeros
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pv[i] = P_KC && pc >= left ? OOB_OFFSET : pv0[i];
      qv[i] = Q_KC && qc >= left ? OOB_OFFSET : qv0[i];
    }
  };
  auto set_bytes = [&](const BigTile& w) {  // KS: bytes that may be read
    const int l = max(min(left, 64), 0);
    if (!P_KC) pbytes = max((l * a.N - w.n0) * 2, 0);
    if (!Q_KC) qbytes = max((l * a.M - w.m0) * 2, 0);
  };
  auto point_at = [&](const BigTile& w) {  // a tile's first stage
    if (KIND == R_TN) {
      left = w.rows;
      pat = (const char*)(a.P + w.row0 * a.N + w.n0);
      qat = (const char*)(a.Q + w.row0 * a.M + w.m0);
    } else {
      left = w.e == a.E ? 0 : a.K;  // rows of nobody: all zeros
      qat = (const char*)(a.Q + w.row0 * a.K);
      qbytes = left > 0 ? w.rows * a.K * 2 : 0;
      pat = (const char*)(a.P + (long)w.e * a.K * a.N + (P_KC ? (long)w.n0 * a.K : w.n0));
      pbytes = left > 0 ? min(a.N - w.n0, BN) * a.K * 2 : 0;
    }
    set_bytes(w);
    if ((P_KC || Q_KC) && a.K % 64 != 0) mask_offsets();
  };
  auto point_on = [&](const BigTile& w) {
    left -= 64;
    pat += pstep;
    qat += qstep;
    if (P_KC) pbytes -= 128;
    if (Q_KC) qbytes -= 128;
    if (left < 64) {
      set_bytes(w);
      if (P_KC || Q_KC) mask_offsets();
    }
  };
  // a stage's loads: 8 of P, 8 of Q
  auto load_to = [&](auto x) {
    constexpr int X = decltype(x)::value;
    lds_load_to<(X < 8 ? 0 : BSLOT * 2) + (X & 7) * BT * 16>(to);
  };
  auto load_go = [&](auto x, i32x4 p, i32x4 q) {
    constexpr int X = decltype(x)::value;
    if constexpr (X < 8) lds_load_go(p, pv[X]);
    else lds_load_go(q, qv[X - 8]);
  };
  auto load = [&](auto x, i32x4 p, i32x4 q) {
    load_to(x);
    asm volatile("s_nop 0");
    load_go(x, p, q);
  };
  auto load_all = [&]() {
    const i32x4 p = settled_rsrc(pat, pbytes), q = settled_rsrc(qat, qbytes);
    each<16>([&](auto x) { load(x, p, q); });
  };
  // a tile's bias, with its first stage, by the first wave: loads are up to two tiles ahead
  auto stage_bias = [&](const BigTile& w, int turn) {
    if (KIND == R_NT && a.bias != nullptr && wave == 0) {
      const int size = a.bias_bf16 ? 2 : 4;
      const char* at = (const char*)a.bias + ((long)w.e * a.N + w.n0) * size;
      const i32x4 r = settled_rsrc(at, w.e == a.E ? 0 : min(a.N - w.n0, BN) * size);
      lds_load16(r, lane * 16, bias0 + (turn & 3) * (BN * 4));
    }
  };

  f32x4 acc[8][8], dbacc[4];
  auto begin = [&](int turn) {  // at the bias of a lane's 8 columns
    float bias[8] = {};
    if (P_KC && a.bias != nullptr) {
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int n = wn * 128 + l15 * 8 + x;
        bias[x] = a.bias_bf16 ? bf2f(((const __bf16*)bias_lds[turn & 3])[n]) : bias_lds[turn & 3][n];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[i][j] = {bias[i], bias[i], bias[i], bias[i]};
        pin_acc(acc[i][j]);
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dbacc[j] = {0.f, 0.f, 0.f, 0.f};
      if (KIND == R_TN) pin_vgpr(dbacc[j]);
    }
    settle();
  };

  // P's fragment i, lane l15 of KC: row 128 wn + 8 l15 + i, so that a lane has 8 neighbouring
  // outputs of a row and 16 lanes the wave's 128. KS: column 128 wn + 16 i + l15.
  // Q's fragment j: rows 32 j + 16 wm + l15, so that both halves of the waves have work in a
  // tile of few rows. The lanes' addresses are kept, and move between the two places by one
  // addition a stage: KC has one for each contraction half, KS one for each column base.
  const unsigned smem0 = lds_addr(smem);
  constexpr int PA = P_KC ? 2 : 8, QA = Q_KC ? 2 : 4;
  unsigned pa[PA], qa[QA];
#pragma unroll
  for (int x = 0; x < PA; ++x) {
    if (P_KC) {
      const int r = wn * 128 + (l15 >> 2) * 8 + (l15 & 3);
      pa[x] = smem0 + (r * 64 + ((x * 4 + g) ^ kc_swz<3>(r)) * 8) * 2;
    } else {
      const int r = g * 8 + (l15 >> 2), col = wn * 128 + x * 16 + 4 * (l15 & 3);
      pa[x] = smem0 + (r * BN + ((col >> 3) ^ ks_swz(r)) * 8 + (col & 7)) * 2;
    }
  }
#pragma unroll
  for (int x = 0; x < QA; ++x) {
    if (Q_KC) {
      const int r = wm * 16 + l15;
      qa[x] = smem0 + BSLOT * 2 + (r * 64 + ((x * 4 + g) ^ kc_swz<2>(r)) * 8) * 2;
    } else {
      const int r = g * 8 + (l15 >> 2), col = x * 32 + wm * 16 + 4 * (l15 & 3);
      qa[x] = smem0 + BSLOT * 2 + (r * 128 + ((col >> 3) ^ ks_swz(r)) * 8 + (col & 7)) * 2;
    }
  }
  auto read_p = [&](int kk, int i) {
    if (P_KC) return lds_read16(pa[kk], ((i >> 1) * 32 + (i & 1) * 4) * 128);
    return lds_read_tr(pa[i % PA], kk * 32 * BN * 2, 4 * BN * 2);
  };
  auto read_q = [&](int kk, int j) {
    if (Q_KC) return lds_read16(qa[kk], j * 32 * 128);
    return lds_read_tr(qa[j % QA], (j / 4) * BSLOT + kk * 32 * 128 * 2, 4 * 128 * 2);
  };
  int hop = 2 * BSLOT * 2, load_hop = hop;
  auto other_place = [&]() {
#pragma unroll
    for (int x = 0; x < PA; ++x) pa[x] += hop;
#pragma unroll
    for (int x = 0; x < QA; ++x) qa[x] += hop;
    hop = -hop;
  };

  // ---- epilogue: 256 bytes of 4 rows in a store. (64 bytes of 16 are written at 3.6 TB/s
  // where these take 4.3: dW of 1024 experts of 32 rows, 2048 x 512, 590 us and 500.) KC has
  // its results so: rows 4g .. 4g + 3 of Q's fragment, 8 columns. KS, with row l15 and columns
  // 4g .. 4g + 3 of each fragment, turns them in LDS. Every lane stores every time, to a place
  // past the descriptor's end where it has nothing: the wait counts on STORES of them.
  constexpr bool F32 = KIND == R_TN && EPI != R_BF16;
  constexpr int STORES = F32 || (KIND == R_NT && EPI == R_GELU_DER) ? 52 : 32;  // of 64: the counter goes to 63
  auto finish = [&](const BigTile& w) {
    int l15 = lane & 15, g = lane >> 4;
    asm volatile("" : "+v"(l15), "+v"(g));  // offsets made from these are not kept through the loop
    settle();
    const long base = (KIND == R_TN ? (long)w.out * a.M + w.m0 : w.row0) * a.N + w.n0;
    const auto rc = __builtin_amdgcn_make_buffer_rsrc((char*)a.C + base * (F32 ? 4 : 2), (short)0, 0x7fffffff, 0x00027000);
    const auto rd = __builtin_amdgcn_make_buffer_rsrc((char*)a.der + base * 2, (short)0, 0x7fffffff, 0x00027000);
    const bool lines = (a.N * (F32 ? 4 : 2)) % 128 == 0;
    const int ncols = a.N - w.n0, nrows = KIND != R_TN || (EPI == R_F32_ACC && w.rows == 0) ? w.rows : a.M - w.m0;
    if (KIND == R_TN && EPI != R_F32_ACC && w.rows == 0) {
      // No rows: the expert's zeros as they lie, whole lines whatever N is, as many stores as a
      // tile has (186 experts of 2968 x 1392, 4 of them with rows: 591 us by tiles)
      constexpr int CHUNK = BM * BN * (F32 ? 4 : 2);
      const long size = (long)a.M * a.N * (F32 ? 4 : 2), from = (long)w.q * CHUNK;
      const int here = (int)max(min(size - from, (long)CHUNK), 0l);
      const auto rz = __builtin_amdgcn_make_buffer_rsrc((char*)a.C + w.out * size + from, (short)0,
                                                        here, 0x00027000);
#pragma unroll
      for (int i = 0; i < CHUNK / (BT * 16); ++i)
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{0, 0, 0, 0}, rz, (i * BT + wave * 64 + lane) * 16, 0, 2);
    } else {
      char* const turn_row = turn_lds[P_KC ? 0 : wave] + l15 * OUT_ROW;  // written by rows, 4 columns a lane
      char* const turn_at = turn_lds[P_KC ? 0 : wave] + g * OUT_ROW + l15 * 16;
      // Slopes, or what sums are added to, of BATCH fragments at once: a load behind stores comes
      // no earlier than these end (dx times slope, 256 experts of 1024 rows, 1024 -> 4096: 2607 us
      // one by one, 2442 by 2, 2395 by 4, 2423 by 8).
      constexpr bool ADDS = KIND == R_TN && EPI == R_F32_ACC;
      constexpr int BATCH = ADDS ? 2 : 4;
      f32x4 sums[ADDS ? BATCH : 1][2][4];
      u32x4 slope[KIND == R_NN && EPI == R_MUL ? BATCH : 1][4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (KIND == R_NN && EPI == R_MUL && j % BATCH == 0) {
#pragma unroll
          for (int b = 0; b < BATCH; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = (j + b) * 32 + wm * 16 + 4 * k + g, n = wn * 128 + l15 * 8;
              const unsigned off = r < nrows && n < ncols ? (unsigned)(r * a.N + n) * 2 : OOB_OFFSET;
              slope[b][k] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rd, off, 0, 0));
            }
          __builtin_amdgcn_sched_barrier(0);
        }
        if (ADDS && j % BATCH == 0) {
#pragma unroll
          for (int b = 0; b < BATCH * 8; ++b) {
            const int r = (j + b / 8) * 32 + wm * 16 + 4 * (b % 4) + g, n = wn * 128 + b / 4 % 2 * 64 + l15 * 4;
            const unsigned off = r < nrows && n < ncols ? (unsigned)(r * a.N + n) * 4 : OOB_OFFSET;
            sums[b / 8][b / 4 % 2][b % 4] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rc, off, 0, 0));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) pin_acc(acc[i][j]);
        const int r0 = j * 32 + wm * 16;
        if (P_KC) {
          const int n = wn * 128 + l15 * 8;
          unsigned off[4];
          bf16x8 o[4];
          f16x8 d[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = r0 + 4 * g + x;
            off[x] = r < nrows && n < ncols ? (unsigned)(r * a.N + n) * 2 : OOB_OFFSET;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float v = acc[i][j][x];
              if (EPI == R_GELU) {
                o[x][i] = f2bf(gelu_of(v));
              } else if (EPI == R_GELU_DER) {
                float y, s;
                gelu_and_slope(v, &y, &s);
                o[x][i] = f2bf(y);
                d[x][i] = (_Float16)s;
              } else {
                o[x][i] = f2bf(v);
              }
            }
          }
          store4(o, rc, off, lines);
          if (EPI == R_GELU_DER) store4(d, rd, off, lines);
        } else {
          if (EPI == R_MUL && KIND == R_NN) {  // to where its products go
#pragma unroll
            for (int k = 0; k < 4; ++k) *(u32x4*)(turn_at + 4 * k * OUT_ROW) = slope[j % BATCH][k];
            asm volatile("" ::: "memory");
          }
#pragma unroll
          for (int h = 0; h < (F32 ? 2 : 1); ++h) {  // 256 bytes: 64 numbers of 32 bits or 128 of 16
            if (F32) {
#pragma unroll
              for (int i = 0; i < 4; ++i) *(f32x4*)(turn_row + (i * 16 + g * 4) * 4) = acc[4 * h + i][j];
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                bf16x4 o;
                if (EPI != R_MUL) {
#pragma unroll
                  for (int x = 0; x < 4; ++x) o[x] = f2bf(acc[i][j][x]);
                } else {
                  const f16x4 d = *(const f16x4*)(turn_row + (i * 16 + g * 4) * 2);
#pragma unroll
                  for (int x = 0; x < 4; ++x) o[x] = f2bf(acc[i][j][x] * (float)d[x]);
                }
                *(bf16x4*)(turn_row + (i * 16 + g * 4) * 2) = o;
              }
            }
            const int n = wn * 128 + h * 64 + l15 * (F32 ? 4 : 8);
            f32x4 turned[4];
            // LDS works in the order of a wave's instructions; the compiler, who sees one lane, is to keep it
            asm volatile("" ::: "memory");
#pragma unroll
            for (int k = 0; k < 4; ++k) turned[k] = *(const f32x4*)(turn_at + 4 * k * OUT_ROW);
            asm volatile("" ::: "memory");
            unsigned off[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = r0 + 4 * k + g;
              off[k] = r < nrows && n < ncols ? (unsigned)(r * a.N + n) * (F32 ? 4 : 2) : OOB_OFFSET;
              if (ADDS) turned[k] += sums[j % BATCH][h][k];
            }
            store4(turned, rc, off, lines);
          }
        }
      }
    }
    if (KIND == R_TN && a.db != nullptr && w.n0 == 0 && g == 0) {  // all 16 D rows hold the same sums
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        pin_vgpr(dbacc[x]);
        const int m = w.m0 + (4 * wn + x) * 32 + wm * 16 + l15;
        if (m < a.M) {
          const long at = (long)w.out * a.M + m;
          if (a.bias_bf16) ((__bf16*)a.db)[at] = f2bf(dbacc[x][0]);
          else ((float*)a.db)[at] = (EPI == R_F32_ACC ? ((float*)a.db)[at] : 0.f) + dbacc[x][0];
        }
      }
    }
  };

  if (mine >= tiles) return;
  // dW back and forth through the blocks, since a round's first tiles are its longest where
  // experts come by their rows.
  auto tile_of = [&](int turn) { return turn * stride + (KIND == R_TN && turn & 1 ? stride - 1 - mine : mine); };
  int loading = mine, lt = 0, lturn = 0;  // the tile and stage that are loaded next
  BigTile lw = decode(loading), w = lw;
  // past the last tile, nothing is loaded
  auto next_stage = [&]() {
    to += load_hop;
    load_hop = -load_hop;
    if (loading >= tiles) {
      pbytes = qbytes = 0;
      return;
    }
    if (++lt < lw.steps) {
      point_on(lw);
    } else {
      lt = 0;
      loading = tile_of(++lturn);
      if (loading < tiles) {
        lw = decode(loading);
        point_at(lw);
        stage_bias(lw, lturn);
      } else {
        pbytes = qbytes = 0;
      }
    }
  };

  bf16x8 p0[8], q0[8], p1[8], q1[8], ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.0f;
  asm volatile("" : "+v"(ones));  // not made anew before each product
  // A quarter of a stage: 32 MFMAs. Behind the first 16, every other time, one of 8 LDS
  // reads; `loads` loads from `load0` on, five MFMAs apart, the first behind the fourth: five
  // instructions and more behind its descriptor (settled_rsrc). More than three instructions
  // behind one MFMA keep the next one waiting. The products of the second rows (j0 = 4) are
  // left out where a tile has none. (Left out by 64 rows instead of 128 they cost more
  // branches than they save: 256 experts of 1024 rows in the mean, 1024 -> 4096, 2068 us and
  // 2043.)
  auto quarter = [&](const bf16x8(&p)[8], const bf16x8(&q)[8], auto j0_, bool there, bool with_db, auto load0_,
                     auto loads_, auto read) {
    constexpr int j0 = decltype(j0_)::value, load0 = decltype(load0_)::value, loads = decltype(loads_)::value;
    i32x4 rp{}, rq{};
    if constexpr (load0 < 8 && loads > 0) {
      rp = make_rsrc(pat, pbytes);
      asm volatile("" : "+s"(rp));
    }
    if constexpr (load0 + loads > 8) {
      rq = make_rsrc(qat, qbytes);
      asm volatile("" : "+s"(rq));
    }
    __builtin_amdgcn_sched_barrier(0);
    if (j0 == 0 || there) {
      each<32>([&](auto x) {
        constexpr int X = decltype(x)::value, i = X % 8, j = j0 + X / 8, n = X / 5;
        if constexpr (X % 5 == 3 && n < loads) load_to(number<load0 + n>());
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (P_KC) mfma_acc(acc[i][j], q[j], p[i]);
        else mfma_acc(acc[i][j], p[i], q[j]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (X % 5 == 3 && n < loads) load_go(number<load0 + n>(), rp, rq);
        if constexpr (X < 16 && X % 2 == 0) read(number<X / 2>());
        __builtin_amdgcn_sched_barrier(0);
      });
      if (KIND == R_TN && with_db && wn == j0 / 4) {  // db: the sums of Q's columns
#pragma unroll
        for (int j = 0; j < 4; ++j) mfma_vgpr(dbacc[j], ones, q[j0 + j]);
      }
    } else {
      each<8>(read);  // these stand between the descriptor and the loads
      __builtin_amdgcn_sched_barrier(0);
      each<loads>([&](auto x) { load(number<load0 + decltype(x)::value>(), rp, rq); });
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  const number<0> first_rows;
  const number<4> last_rows;

#pragma unroll
  for (int i = 0; i < 8; ++i) {
    pv[i] = pv0[i];
    qv[i] = qv0[i];
  }
  stage_bias(lw, 0);
  point_at(lw);
  load_all();
  next_stage();
  load_all();
  wait_and_barrier<16>();
  each<8>([&](auto x) { p0[decltype(x)::value] = read_p(0, decltype(x)::value); });
  each<8>([&](auto x) { q0[decltype(x)::value] = read_q(0, decltype(x)::value); });
  next_stage();
  bool stored = false;  // the last tile's stores lie between this stage and the one before
  for (int at = mine, turn = 0; at < tiles; at = tile_of(++turn)) {
    if (turn > 0) w = decode(at);
    const bool both = KIND == R_TN || w.rows > 128;  // the tile's second half of rows is there
    const bool with_db = KIND == R_TN && a.db != nullptr && w.n0 == 0;
    begin(turn);
    for (int t = 0; t < w.steps; ++t) {
      // Each quarter reads 8 fragments, early, for the next but one: at 128 bytes a cycle
      // these and what comes in take three quarters of it.
      quarter(p0, q0, first_rows, true, with_db, number<0>(), number<0>(),
              [&](auto x) { p1[decltype(x)::value] = read_p(1, decltype(x)::value); });
      wait_reads_and_barrier();  // nobody reads this stage's P any more
      // A CU takes 64 bytes a cycle: a stage's loads keep it busy for half a stage, and
      // where they come faster the wave stands at the next one and multiplies nothing.
      quarter(p0, q0, last_rows, both, with_db, number<0>(), number<5>(),
              [&](auto x) { q1[decltype(x)::value] = read_q(1, decltype(x)::value); });
      other_place();
      // nor its Q, and P of the next stage has landed
      if (stored) wait_and_barrier<(13 + STORES < 63 ? 13 + STORES : 63)>();
      else wait_and_barrier<13>();
      quarter(p1, q1, first_rows, true, with_db, number<5>(), number<6>(),
              [&](auto x) { p0[decltype(x)::value] = read_p(0, decltype(x)::value); });
      // and its Q
      if (stored) wait_loads_and_barrier<11 + STORES>();
      else wait_loads_and_barrier<11>();
      stored = false;
      quarter(p1, q1, last_rows, both, with_db, number<11>(), number<5>(),
              [&](auto x) { q0[decltype(x)::value] = read_q(0, decltype(x)::value); });
      next_stage();
    }
    finish(w);
    stored = true;
  }
  // nothing may come into this block's LDS once it is another's
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}

// 16-row tiles where experts have a row or none: of 256 experts, 1024 -> 4096, 4 rows take 12
// us so and 49 in 128-row tiles, 128 rows 158 and 168, 1024 rows 422 and 361. And for small
// products, which leave most CUs idle in 128-row tiles: by rows and experts times outputs (8
// experts of 128 rows, 256 -> 256, 18432: 5.3 us and 10; 12 of 166, 136 -> 328, 44895: 8.2 and
// 9.8; 8 of 128, 256 -> 1024, 73728: 15 and 10), as long as the weights, read anew for every
// 16 rows, take no longer than a contraction in parts (4 of 64 rows, 1024 -> 1024, 21 million:
// 12 and 15; 4 of 128, 38 million: 21 and 19; 4 of 16, 4096 -> 4096, 134 million: 41 and 28).
static bool few_rows(long R, int E, int N, int K) {
  const long outputs = (R / FR + E) * N;
  return R <= E || (outputs <= 49152 && outputs * K <= 32 << 20);
}

template <int EPI>
static void launch_few(const RaggedArgs& a, hipStream_t stream) {
  const long most = a.R < a.R / FR + a.E + 1 ? a.R : a.R / FR + a.E + 1;
  const int groups = cdiv(a.N, FR);
  // outputs a block, one group of 16 after the other: looking up its tile is as long as one
  const int per = (int)(most * groups <= 8192 ? 1 : most * groups <= 32768 ? 4 : 8);
  hipLaunchKernelGGL((ragged_few_kernel<EPI>), dim3(cdiv(groups, per), (unsigned)most), dim3(256), 0, stream, a,
                     per);
}

// Weights larger than the last cache (256 MB) are gone before the next call, and where
// experts have few rows each is read once or twice: such loads leave L2 to the rows. 1024
// experts of 32 rows, 2048 -> 512: 434 us, 467 without; 256 of 8, 1024 -> 4096: 334 and 360,
// its dx 346 and 383. Smaller weights lose by it: 64 of 1024 x 1024, 64 rows each, 42 and 39.
static bool read_once(int E, int N, int K) { return (long)E * N * K * 2 > (256l << 20); }

// Rows from the parts' sums, in the parts' order, and what else belongs to them
template <int EPI>
__launch_bounds__(256) __global__ void ragged_join_rows_kernel(RaggedArgs a, const float* __restrict__ part) {
  const long n = a.R * a.N, i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 v = *(const f32x4*)(part + i);
  for (int p = 1; p < a.splits; ++p) v += *(const f32x4*)(part + p * n + i);
  if (a.bias != nullptr) {
    const long row = i / a.N;
    int e = 0;  // the last group that starts at or before the row has it
    for (int end = a.E; e < end;) {
      const int mid = (e + end + 1) >> 1;
      if (a.offsets[mid] <= row) e = mid;
      else end = mid - 1;
    }
    if (e < a.E) {
      const long at = (long)e * a.N + i % a.N;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        v[x] += a.bias_bf16 ? bf2f(((const __bf16*)a.bias)[at + x]) : ((const float*)a.bias)[at + x];
    }
  }
  bf16x4 o;
  f16x4 d;
  if (EPI == R_MUL) d = *(const f16x4*)(a.der + i);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (EPI == R_GELU_DER) {
      float y, s;
      gelu_and_slope(v[x], &y, &s);
      o[x] = f2bf(y);
      d[x] = (_Float16)s;
    } else {
      o[x] = f2bf(EPI == R_GELU ? gelu_of(v[x]) : EPI == R_MUL ? v[x] * (float)d[x] : v[x]);
    }
  }
  *(bf16x4*)((__bf16*)a.C + i) = o;
  if (EPI == R_GELU_DER) *(f16x4*)(a.der + i) = d;
}

// Parts of the contraction where there are fewer tiles than CUs, a microsecond for each 64
// steps; of few rows, whose sums are small, for two blocks a CU. 4 experts of 32 rows, dx
// 1024 <- 4096: 77 us in one part, 20 in 12 and 25; 4 of 64 rows, 4096 -> 4096: 76, 47 in 2, 42
// in 5; 8 of 512 rows, 1024 -> 1024, 29 us, 48 in 3 parts.
extern "C" int lah_ragged_parts(long R, int E, int N, int K, bool forward) {
  if (forward && few_rows(R, E, N, K)) return 1;
  const long tiles = (R < R / RBM + E ? R : R / RBM + E) * ((N + RBN - 1) / RBN), most = (K + 63) / 64 / 4;
  const long s = (R <= 512 ? 512 : 256) / (tiles < 1 ? 1 : tiles);
  return (int)(s < most ? (s < 1 ? 1 : s) : most < 1 ? 1 : most);
}

template <int KIND, int EPI>
static void launch_rows(const RaggedArgs& a, void* table, void* work, hipStream_t stream) {
  if constexpr (KIND == R_NT)
    if (few_rows(a.R, a.E, a.N, a.K)) return launch_few<EPI>(a, stream);
  if (table != nullptr) {
    hipLaunchKernelGGL(ragged_tiles_kernel, dim3(1), dim3(1024), 0, stream, a.offsets, a.E, a.R, (int4*)table);
    const long most = (a.R / BM + a.E + 1) * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL((ragged_big_kernel<KIND, EPI>), dim3((unsigned)(most < 256 ? most : 256)), dim3(BT), 0,
                       stream, a, (const int4*)table);
    return;
  }
  const unsigned tiles = (unsigned)((a.R / RBM + a.E + 1) * ((a.N + RBN - 1) / RBN));
  if (a.splits > 1) {
    RaggedArgs part = a;
    part.C = work;
    hipLaunchKernelGGL((ragged_rows_kernel<KIND, R_PART>), dim3(tiles, a.splits), dim3(RT), 0, stream, part);
    hipLaunchKernelGGL((ragged_join_rows_kernel<EPI>), dim3((unsigned)((a.R * a.N / 4 + 255) / 256)), dim3(256), 0,
                       stream, a, (const float*)work);
    return;
  }
  hipLaunchKernelGGL((ragged_rows_kernel<KIND, EPI>), dim3(tiles), dim3(RT), 0, stream, a);
}

// dW and db from the parts' sums, in the parts' order
template <int OUT>
__launch_bounds__(256) __global__ void ragged_join_kernel(const float* __restrict__ part, int splits, long n,
                                                          void* __restrict__ out) {
  const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 sum = *(const f32x4*)(part + i);
  for (int s = 1; s < splits; ++s) sum += *(const f32x4*)(part + s * n + i);
  if (OUT == R_BF16) {
    bf16x4 o;
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] = f2bf(sum[x]);
    *(bf16x4*)((__bf16*)out + i) = o;
  } else {
    float* c = (float*)out + i;
    *(f32x4*)c = OUT == R_F32_ACC ? *(const f32x4*)c + sum : sum;
  }
}

static void join(const float* part, int splits, long n, void* out, int kind, hipStream_t stream) {
  const dim3 grid((unsigned)((n / 4 + 255) / 256)), block(256);
  if (kind == R_BF16) hipLaunchKernelGGL((ragged_join_kernel<R_BF16>), grid, block, 0, stream, part, splits, n, out);
  else if (kind == R_F32_ACC) hipLaunchKernelGGL((ragged_join_kernel<R_F32_ACC>), grid, block, 0, stream, part, splits, n, out);
  else hipLaunchKernelGGL((ragged_join_kernel<R_F32>), grid, block, 0, stream, part, splits, n, out);
}

static long weight_tiles(int E, int N, int M) { return (long)E * ((M + BM - 1) / BM) * ((N + BN - 1) / BN); }

template <int OUT>
static void launch_weights(const RaggedArgs& a, const int4* table, hipStream_t stream) {
  const long tiles = a.splits * weight_tiles(a.E, a.N, a.M);
  hipLaunchKernelGGL((ragged_big_kernel<R_TN, OUT>), dim3((unsigned)(tiles < 256 ? tiles : 256)), dim3(BT), 0,
                     stream, a, table);
}

// order[i] = the expert with the i'th most rows, the lower one of two as large
#define ORDERED 4096  // experts at most
__launch_bounds__(256) __global__ void ragged_order_kernel(const int* __restrict__ offsets, int E, long R,
                                                           int* __restrict__ order) {
  __shared__ __attribute__((aligned(16))) int rows[ORDERED];
  const int Ep = (E + 3) & ~3;
  for (int e = threadIdx.x; e < Ep; e += 256) {
    const long lo = e == 0 || e >= E ? 0 : min((long)max(offsets[e], 0), R);
    rows[e] = e < E ? (int)(min(max((long)offsets[e + 1], lo), R) - lo) : -1;
  }
  __syncthreads();
  const int mine = blockIdx.x * 256 + threadIdx.x;
  if (mine >= E) return;
  const int n = rows[mine];
  int rank = 0;
  for (int e = 0; e < Ep; e += 4) {
    const i32x4 v = *(const i32x4*)(rows + e);
#pragma unroll
    for (int x = 0; x < 4; ++x) rank += v[x] > n || (v[x] == n && e + x < mine);
  }
  order[rank] = mine;
}

// Lists for experts with very different rows. Tiles are as long as their expert's rows, L of
// which are half of what a CU has to do in all. Experts of more than that come first, in pieces
// of L with sums of their own, where the largest has over 4 L; else those of more than 2 L; the
// others come whole and by their rows: pieces[0] = {number, experts}, pieces[1 + i] = {expert, first row,
// rows, i}, joins[k] = {expert, its first piece, pieces}; whole[0] = {number}, whole[1 + i] =
// {expert, first row, rows, expert}.
__launch_bounds__(1024) __global__ void ragged_pieces_kernel(const int* __restrict__ offsets, int E, long R, long L,
                                                             int room, const int* __restrict__ order,
                                                             int4* __restrict__ pieces, int4* __restrict__ joins,
                                                             int4* __restrict__ whole) {
  __shared__ int wsum[16][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PER = ORDERED / 1024;
  int es[PER], c[PER], at = 0, large = 0;
  long lo[PER], rows[PER];
  const int e0 = order[0];
  const long lo0 = e0 == 0 ? 0 : min((long)max(offsets[e0], 0), R);
  const long whole_rows = min(max((long)offsets[e0 + 1], lo0), R) - lo0 > 4 * L ? L : 2 * L;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid * PER + j;
    c[j] = 0;
    if (i >= E) continue;
    es[j] = order[i];
    lo[j] = es[j] == 0 ? 0 : min((long)max(offsets[es[j]], 0), R);
    rows[j] = min(max((long)offsets[es[j] + 1], lo[j]), R) - lo[j];
    if (rows[j] > whole_rows) c[j] = (int)((rows[j] + L - 1) / L);
    at += c[j];
    large += c[j] > 0;
  }
  int inc = at, linc = large;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(inc, d, 64), u = __shfl_up(linc, d, 64);
    if (lane >= d) inc += v, linc += u;
  }
  if (lane == 63) wsum[wave][0] = inc, wsum[wave][1] = linc;
  __syncthreads();
  int first = inc - at, total = 0, most = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    first += w < wave ? wsum[w][0] : 0;
    total += wsum[w][0];
    most += wsum[w][1];
  }
  if (tid == 0) {
    pieces[0] = make_int4(min(total, room), most, 0, 0);
    whole[0] = make_int4(E - most, 0, 0, 0);
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = tid * PER + j;
    if (i >= E) continue;
    if (c[j] == 0) {  // by rows: the large ones are in front
      whole[1 + i - most] = make_int4(es[j], (int)lo[j], (int)rows[j], es[j]);
      continue;
    }
    // more pieces than there is room for: only where offsets do not ascend
    const int n = max(min(c[j], room - first), 0);
    if (i < room) joins[i] = make_int4(es[j], first, n, 0);
    for (int p = 0; p < n; ++p)
      pieces[1 + first + p] = make_int4(es[j], (int)(lo[j] + p * L), (int)min(rows[j] - p * L, L), first + p);
    first += c[j];
  }
}

// dW and db of the experts in pieces, from the pieces' sums, in order
template <int OUT>
__launch_bounds__(256) __global__ void ragged_join_pieces_kernel(RaggedArgs a, const int4* __restrict__ pieces,
                                                                 const int4* __restrict__ joins, int room,
                                                                 const float* __restrict__ part) {
  if ((int)blockIdx.y >= pieces[0].y) return;
  const int4 t = joins[blockIdx.y];
  const long n = (long)a.M * a.N, i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n + (a.db != nullptr ? a.M : 0) || t.z == 0) return;
  const bool is_db = i >= n;
  const float* from = is_db ? part + room * n + (long)t.y * a.M + (i - n) : part + t.y * n + i;
  f32x4 sum = *(const f32x4*)from;
  for (int p = 1; p < t.z; ++p) sum += *(const f32x4*)(from + p * (is_db ? a.M : n));
  if (is_db ? a.bias_bf16 != 0 : OUT == R_BF16) {
    bf16x4 o;
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] = f2bf(sum[x]);
    *(bf16x4*)(is_db ? (__bf16*)a.db + (long)t.x * a.M + (i - n) : (__bf16*)a.C + t.x * n + i) = o;
  } else {
    float* c = is_db ? (float*)a.db + (long)t.x * a.M + (i - n) : (float*)a.C + t.x * n + i;
    *(f32x4*)c = OUT == R_F32_ACC ? *(const f32x4*)c + sum : sum;
  }
}

// The work of dW, in bytes: sums of parts (splits > 1), or lists and sums of pieces
// (where L > 0), or nothing.
struct WeightWork {
  int splits;
  long L;     // rows a piece
  int room;   // pieces at most
  long bytes, sums;  // in all; where the sums begin
};
// int4 entries a table of M-tiles needs
extern "C" long lah_ragged_tiles_room(long R, int E) { return R / BM + E + 2; }

// table: room for the M-tiles where the large tiles are to be used, or null. work: fp32 room for
// parts * R * N, if there are more than one
extern "C" void lah_ragged_nt(const void* x, const void* w, void* y, const void* offsets,
                              const void* bias, int bias_bf16, void* der, long R, int E, int N,
                              int K, int epi, void* table, int parts, void* work, hipStream_t stream) {
  RaggedArgs a{(const __bf16*)w, (const __bf16*)x, y, (const int*)offsets, bias, (_Float16*)der,
               nullptr, R, E, N, 0, K, bias_bf16, parts, read_once(E, N, K)};
  if (epi == R_GELU_DER) launch_rows<R_NT, R_GELU_DER>(a, table, work, stream);
  else if (epi == R_GELU) launch_rows<R_NT, R_GELU>(a, table, work, stream);
  else launch_rows<R_NT, R_PLAIN>(a, table, work, stream);
}

// dx[r] = W[e]^T d[r] (times der[r], if given): W [E, K, N], d [R, K], out [R, N]
extern "C" void lah_ragged_nn(const void* d, const void* w, void* out, const void* offsets,
                              void* der, long R, int E, int N, int K, void* table, int parts, void* work,
                              hipStream_t stream) {
  RaggedArgs a{(const __bf16*)w, (const __bf16*)d, out, (const int*)offsets, nullptr,
               (_Float16*)der, nullptr, R, E, N, 0, K, 0, parts, read_once(E, N, K)};
  if (der != nullptr) launch_rows<R_NN, R_MUL>(a, table, work, stream);
  else launch_rows<R_NN, R_PLAIN>(a, table, work, stream);
}

// Parts of each expert's rows, where there are fewer tiles than CUs: tiles for all of them, or
// for each twice where there are many, since experts' rows are not alike; at least 4 stages a
// part in the mean. 2 experts of 131072 rows, 512 x 512 (8 tiles): 2655 us in one part, 146 in
// 32, 221 in 64; 8 with 13123 of 32768 rows, 1024 x 1024 (128 tiles), 272 in one, 160 in 2, 117
// in 4, 171 in 8; 16 of 1024 rows, 512 x 512, 31 in one and 37 in 4.
static int splits_of(long R, int E, int N, int M) {
  const long tiles = weight_tiles(E, N, M), most = R / E / 256;
  const long s = tiles < 64 ? 256 / tiles : tiles < 256 ? 512 / tiles : 1;
  return (int)(s < most ? s : most < 1 ? 1 : most);
}

// Lists by rows where there are many tiles and rows, pieces of half a CU's share and at
// least 16 stages. 256 experts with 15358 rows down to none, 262144 in all, 4096 x 1024: 2403 us
// in the experts' order, 2254 back and forth, 2167 by rows. 145 experts, one with 15082 of 99929
// rows (7 L), 248 x 2632: 428 us by rows, 287 in pieces of all above L, 319 of all above 2 L;
// 128, 12745 of 131072 (3.1 L), 1024 x 1024: 386, 400 and 335; 64, 10002 of 262144 (1.2 L): 490,
// 561 and 490. Few rows are bound by the stores, which the longer tiles' products then no
// longer hide: 1024 experts, 32768 rows, 1280 down to none, 512 x 2048: 404 us and 450 by rows.
static WeightWork weight_work(long R, int E, int N, int M) {
  WeightWork w{splits_of(R, E, N, M), 0, 0, 0, 0};
  const long one = (long)M * (N + 1) * 4, tiles = weight_tiles(1, N, M);
  if (w.splits > 1) {
    w.bytes = w.splits * E * one;
  } else if (E > 1 && E <= ORDERED && R / 256 >= E && tiles * E > 256) {
    const long half = R * tiles / 256 / 2;
    w.L = ((half > 1024 ? half : 1024) + 63) & ~63l;
    w.room = R > w.L ? (int)(2 * R / w.L) + 1 : 0;
    w.sums = ((2l * w.room + E + 2) * 16 + E * 4 + 255) & ~255l;
    w.bytes = w.sums + w.room * one;
  }
  return w;
}

extern "C" long lah_ragged_tn_work(long R, int E, int N, int M) { return weight_work(R, E, N, M).bytes; }

// dw[e] = sum_r d[r] x[r]^T: d [R, M], x [R, N], dw [E, M, N]; db [E, M] or null;
// work: lah_ragged_tn_work bytes
extern "C" void lah_ragged_tn(const void* d, const void* x, void* dw, void* db, int db_bf16,
                              const void* offsets, long R, int E, int N, int M, int out, void* work,
                              hipStream_t stream) {
  const WeightWork need = weight_work(R, E, N, M);
  RaggedArgs a{(const __bf16*)x, (const __bf16*)d, dw, (const int*)offsets, nullptr, nullptr,
               db, R, E, N, M, 0, db_bf16, need.splits, false};
  const long n = (long)M * N;
  if (need.splits > 1) {
    const int splits = need.splits;
    float* db_part = (float*)work + splits * E * n;
    a.C = work;
    a.db = db != nullptr ? db_part : nullptr;
    a.bias_bf16 = 0;
    launch_weights<R_F32>(a, nullptr, stream);
    join((const float*)work, splits, E * n, dw, out, stream);
    if (db != nullptr)
      join(db_part, splits, (long)E * M, db, db_bf16 ? R_BF16 : out == R_F32_ACC ? R_F32_ACC : R_F32, stream);
    return;
  }
  const int4* table = nullptr;
  if (need.L > 0) {
    int4* const pieces = (int4*)work;
    int4* const joins = pieces + need.room + 1;
    int4* const whole = joins + need.room;
    int* const order = (int*)(whole + E + 1);
    float* const part = (float*)((char*)work + need.sums);
    hipLaunchKernelGGL(ragged_order_kernel, dim3(cdiv(E, 256)), dim3(256), 0, stream, a.offsets, E, R, order);
    hipLaunchKernelGGL(ragged_pieces_kernel, dim3(1), dim3(1024), 0, stream, a.offsets, E, R, need.L, need.room,
                       (const int*)order, pieces, joins, whole);
    const dim3 grid((unsigned)((n + M + 1023) / 1024), (unsigned)(R / need.L < E ? R / need.L : E));
    if (grid.y > 0) {  // some may have more than L rows
      RaggedArgs p = a;
      p.C = part;
      p.db = db != nullptr ? part + need.room * n : nullptr;
      p.bias_bf16 = 0;
      launch_weights<R_F32>(p, pieces, stream);
      auto join_pieces = out == R_BF16 ? ragged_join_pieces_kernel<R_BF16>
                         : out == R_F32_ACC ? ragged_join_pieces_kernel<R_F32_ACC> : ragged_join_pieces_kernel<R_F32>;
      hipLaunchKernelGGL(join_pieces, grid, dim3(256), 0, stream, a, (const int4*)pieces, (const int4*)joins,
                         need.room, (const float*)part);
    }
    table = whole;
  }
  if (out == R_BF16) launch_weights<R_BF16>(a, table, stream);
  else if (out == R_F32_ACC) launch_weights<R_F32_ACC>(a, table, stream);
  else launch_weights<R_F32>(a, table, stream);
}

// The group of a slot (find_expert) in two steps of 64: starts grow with the group. Each block
// of the pass below looks for its own, and many have few rows: 4096 groups of 2048 rows, 4096
// columns, 52 us, 345 with find_expert's 65 ballots.
LAH_DEVINL int find_slot(const int* __restrict__ offsets, int E, int slot) {
  const int lane = threadIdx.x & 63;
  auto begun = [&](int e) { return e < E && (e > 0 ? offsets[e] : 0) / RBM + e <= slot; };
  const int base = (__popcll(__ballot(begun(lane * 64))) - 1) * 64;
  const int e = base + __popcll(__ballot(begun(base + lane))) - 1;
  return offsets[E] / RBM + E <= slot ? E : e;  // rows of nobody
}

// dP = dy * slope, rounded to bf16 for the two products that take it, and db, its sums over each
// group's rows as they were before that. A tile is up to 128 rows of one group by 256 columns,
// 8 a lane; where there are fewer columns its lanes take more rows. Its sums go to part[slot],
// and are joined in the slots' order. Or it is a whole group, by 64 columns, and needs no join.
// Rows of nobody are left out: nothing reads their dP. Bound by HBM: dy and the slope in, dP out.
// 262144 rows of 4096: 1230 us with db and without, 6.4 GB at 5.2 TB/s.
enum { S_NONE = 0, S_PART = 1, S_GROUP = 2 };  // sums: none, of a tile, of a group
template <bool WRITE, int SUMS>
__launch_bounds__(256) __global__ void ragged_slope_kernel(RaggedArgs a, const __bf16* __restrict__ dy,
                                                           __bf16* __restrict__ dp, float* __restrict__ part,
                                                           int shift, int tiles) {
  __shared__ __attribute__((aligned(16))) float sums[2048];  // [row lanes][columns]
  const int lanes = 1 << shift, NT = cdiv(a.N, lanes * 8), step = 256 >> shift;
  const int c = threadIdx.x & (lanes - 1), r0 = threadIdx.x >> shift;
  for (int L = blockIdx.x; L < tiles; L += gridDim.x) {
    const int slot = L / NT, n0 = L % NT * lanes * 8, n = n0 + c * 8;
    const int e = SUMS == S_GROUP ? slot : __builtin_amdgcn_readfirstlane(find_slot(a.offsets, a.E, slot));
    if (e < 0 || e >= a.E) continue;
    long lo, hi;
    expert_rows(a, e, &lo, &hi);
    const long row0 = SUMS == S_GROUP ? lo : lo + (long)(slot - (int)(lo / RBM) - e) * RBM;
    if (SUMS != S_GROUP && (row0 < lo || row0 >= hi)) continue;
    const int rows = (int)(SUMS == S_GROUP ? hi - lo : min(hi - row0, (long)RBM));
    float sum[8] = {};
    if (n < a.N) {
      const long at = row0 * a.N + n;
      for (int r = r0; r < rows; r += 4 * step) {  // four rows' loads at once
        bf16x8 y[4];
        f16x8 d[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const bool in = r + u * step < rows;
          y[u] = in ? *(const bf16x8*)(dy + at + (long)(r + u * step) * a.N) : bf16x8{};
          d[u] = in ? *(const f16x8*)(a.der + at + (long)(r + u * step) * a.N) : f16x8{};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          bf16x8 o;
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float v = bf2f(y[u][x]) * (float)d[u][x];
            sum[x] += v;
            o[x] = f2bf(v);
          }
          if (WRITE && r + u * step < rows) *(bf16x8*)(dp + at + (long)(r + u * step) * a.N) = o;
        }
      }
    }
    if (SUMS == S_NONE) continue;
#pragma unroll
    for (int h = 0; h < 8; h += 4)
      *(f32x4*)(sums + (r0 * lanes + c) * 8 + h) = f32x4{sum[h], sum[h + 1], sum[h + 2], sum[h + 3]};
    __syncthreads();
    const int col = threadIdx.x;
    if (col < lanes * 8 && n0 + col < a.N) {
      float all = 0.f;
      for (int r = 0; r < min(step, rows); ++r) all += sums[r * lanes * 8 + col];  // lanes past the rows have none
      const long to = (long)slot * a.N + n0 + col;
      if (SUMS == S_PART) part[to] = all;
      else if (a.bias_bf16) ((__bf16*)a.db)[to] = f2bf(all);
      else ((float*)a.db)[to] = all;
    }
    __syncthreads();  // the next tile's sums
  }
}

// db of each group from its slots' sums, four columns a lane: four quarters of the slots in turn,
// joined in order
__launch_bounds__(256) __global__ void ragged_join_sums_kernel(RaggedArgs a, const float* __restrict__ part, int tiles) {
  __shared__ f32x4 sums[4][64];
  const int c = threadIdx.x & 63, q = threadIdx.x >> 6, NT = cdiv(a.N, 256);
  for (int L = blockIdx.x; L < tiles; L += gridDim.x) {
    const int e = L / NT, n = L % NT * 256 + c * 4;
    long lo, hi;
    expert_rows(a, e, &lo, &hi);
    const int count = (int)((hi - lo + RBM - 1) / RBM);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    if (n < a.N) {
      const float* at = part + ((lo / RBM) + e) * a.N + n;
#pragma unroll 8
      for (int i = q; i < count; i += 4) sum += *(const f32x4*)(at + (long)i * a.N);
    }
    sums[q][c] = sum;
    __syncthreads();
    if (q == 0 && n < a.N) {
      const f32x4 all = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
      const long to = (long)e * a.N + n;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (a.bias_bf16) ((__bf16*)a.db)[to + x] = f2bf(all[x]);
        else ((float*)a.db)[to + x] = all[x];
      }
    }
    __syncthreads();
  }
}

// Whole groups where none can be long: 128 rows are a round of a block, and one more launch is
// as long as a few. 12 groups of 1998 rows, 136 -> 328, forward and backward: 80 us so, 86 joined.
static bool slope_by_group(long R) { return R <= 16 * RBM; }

// fp32 numbers that the slots' sums need room for
extern "C" long lah_ragged_slope_work(long R, int E, int N) {
  return slope_by_group(R) ? 0 : (R / RBM + E + 1) * N;
}

// dp [R, N] = dy * der, or null; db [E, N] or null, with work: lah_ragged_slope_work numbers
extern "C" void lah_ragged_slope(const void* dy, const void* der, void* dp, void* db, int db_bf16,
                                 const void* offsets, long R, int E, int N, void* work, hipStream_t stream) {
  RaggedArgs a{nullptr, nullptr, nullptr, (const int*)offsets, nullptr, (_Float16*)der,
               db, R, E, N, 0, 0, db_bf16, 1, false};
  const bool by_group = db != nullptr && slope_by_group(R);
  int shift = 0;
  while (shift < (by_group ? 3 : 5) && (8 << shift) < N) ++shift;
  // many groups of few rows: more columns a tile
  while (by_group && shift < 5 && (8 << shift) < N && (long)E * cdiv(N, 8 << shift) > 16384) ++shift;
  const long tiles = (by_group ? E : R / RBM + E + 1) * cdiv(N, 8 << shift);
  auto blocks = [](long n) { return dim3((unsigned)(n < 16384 ? n : 16384)); };
  auto kernel = dp == nullptr ? (by_group ? ragged_slope_kernel<false, S_GROUP> : ragged_slope_kernel<false, S_PART>)
                : db == nullptr ? ragged_slope_kernel<true, S_NONE>
                : by_group ? ragged_slope_kernel<true, S_GROUP> : ragged_slope_kernel<true, S_PART>;
  hipLaunchKernelGGL(kernel, blocks(tiles), dim3(256), 0, stream, a, (const __bf16*)dy, (__bf16*)dp, (float*)work,
                     shift, (int)tiles);
  if (db != nullptr && !by_group) {
    const long joined = (long)E * cdiv(N, 256);
    hipLaunchKernelGGL(ragged_join_sums_kernel, blocks(joined), dim3(256), 0, stream, a, (const float*)work,
                       (int)joined);
  }
}
