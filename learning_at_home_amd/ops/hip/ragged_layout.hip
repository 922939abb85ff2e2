// Rows of each expert from the router's choice, for MI355X (gfx950): a stable
// counting sort of the T*k slots by expert, without atomics on the order, so
// that the same choice always gives the same rows.
//
//   offsets[e]  = valid slots of experts below e          [E + 1]
//   order[r]    = slot of row r; -1 from offsets[E] on    [T * k]
//   rows[slot]  = row of the slot; -1 where 0 <= id < E fails
//
// A block takes CH neighbouring slots, a wave 64 at a time, in order. Lanes with
// the same expert find each other by one ballot a bit of the id; the rank of a
// slot is what its wave has counted so far plus its peers in lower lanes. Counts
// of waves (LDS) and of blocks (a table in global memory) are then summed in
// slot order. 4 bytes in, 8 out a slot: what counts is the launches and the
// chain of small steps in each.
#include "common.h"

// 64-slot groups a wave: more blocks while there are few, shorter tables when there are many.
// 98304 slots, 256 experts: 9.6 us by 2 and 12.1 by 4; 65536, 1024: 12.6 and 13.9; 400000, 256:
// 14.9 and 14.4; 1500000, 256: 66 and 43. Up to 4096 one block has all by 4: 7.3 us, 9.2 by 2.
static int layout_groups(long n) { return n > 4096 && n <= 262144 ? 2 : 4; }

template <typename Id>
LAH_DEVINL int id_of(const Id* ids, long s, long n, int E) {
  if (s >= n) return E;
  const Id v = ids[s];
  return v >= 0 && v < (Id)E ? (int)v : E;  // E: no expert
}

// table[b][e] = slots of expert e in block b's chunk
template <typename Id, int CH>
__launch_bounds__(1024) __global__ void layout_count_kernel(const Id* __restrict__ ids, long n, int E,
                                                            int* __restrict__ table) {
  __shared__ int h[4096];
  for (int e = threadIdx.x; e < E; e += 1024) h[e] = 0;
  __syncthreads();
  const long s0 = (long)blockIdx.x * CH;
#pragma unroll
  for (int i = 0; i < CH / 1024; ++i) {
    const int e = id_of(ids, s0 + i * 1024 + threadIdx.x, n, E);
    if (e < E) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += 1024) table[(long)blockIdx.x * E + e] = h[e];
}

// table[b][e] -> sum over blocks before b, in place; table[B][e] = sum over all
__launch_bounds__(64) __global__ void layout_prefix_kernel(int* __restrict__ table, int B, int E) {
  const int e = blockIdx.x * 64 + threadIdx.x;
  if (e >= E) return;
  int sum = 0;
  for (int b0 = 0; b0 < B; b0 += 16) {
    int v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = b0 + j < B ? table[(long)(b0 + j) * E + e] : 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (b0 + j < B) {
        table[(long)(b0 + j) * E + e] = sum;
        sum += v[j];
      }
  }
  table[(long)B * E + e] = sum;
}

enum { LY_ONE = 0, LY_SUM = 1, LY_PREFIX = 2 };  // one block; sums the table itself; prefix kernel ran

template <typename Id, int ECAP, int WAVES, int GROUPS, int MODE>
__launch_bounds__(WAVES * 64) __global__
void layout_place_kernel(const Id* __restrict__ ids, long n, int E, int bits, const int* __restrict__ table,
                         int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ rows) {
  constexpr int T = WAVES * 64, CH = T * GROUPS, PER = ECAP / T > 0 ? ECAP / T : 1;
  __shared__ unsigned short wh[WAVES][ECAP];  // a wave's counts, then those of the waves before it
  __shared__ int start[ECAP], total[ECAP];
  __shared__ int wsum[WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x, B = gridDim.x;
  const long s0 = (long)b * CH + wave * (64 * GROUPS) + lane;

  int id[GROUPS], rank[GROUPS];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) id[i] = id_of(ids, s0 + i * 64, n, E);
  for (int e = lane; e < E; e += 64) wh[wave][e] = 0;
  for (int e = tid; e < E; e += T) start[e] = total[e] = 0;
  __syncthreads();

  if (MODE == LY_SUM) {  // the table's columns, T / E threads each
    const int Ep = E < T ? E : T, groups = T / Ep, grp = tid / Ep;
    if (grp < groups)
      for (int e = tid % Ep; e < E; e += Ep) {
        int before = 0, all = 0;
        for (int q0 = grp; q0 < B; q0 += 16 * groups) {  // 16 loads at once
          int c[16];
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            const int q = q0 + u * groups;
            c[u] = q < B ? table[(long)q * E + e] : 0;
          }
#pragma unroll
          for (int u = 0; u < 16; ++u) {
            all += c[u];
            before += q0 + u * groups < b ? c[u] : 0;
          }
        }
        atomicAdd(&start[e], before);  // whole numbers: the order does not matter
        atomicAdd(&total[e], all);
      }
  } else if (MODE == LY_PREFIX) {
    for (int e = tid; e < E; e += T) {
      start[e] = table[(long)b * E + e];
      total[e] = table[(long)B * E + e];
    }
  }

#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const int e = id[i];
    unsigned long long peers = ~0ull;
    for (int q = 0; q < bits; ++q) {
      const bool on = (e >> q) & 1;
      const unsigned long long m = __ballot(on);
      peers &= on ? m : ~m;
    }
    const int below = __popcll(peers & ((1ull << lane) - 1));
    int had = 0;
    if (e < E) had = wh[wave][e];
    rank[i] = had + below;
    if (e < E && below == 0) wh[wave][e] = (unsigned short)(had + __popcll(peers));
  }
  __syncthreads();

  for (int e = tid; e < E; e += T) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const int c = wh[w][e];
      wh[w][e] = (unsigned short)sum;
      sum += c;
    }
    if (MODE == LY_ONE) total[e] = sum;
  }
  __syncthreads();

  // exclusive sum of total over the experts, PER neighbouring ones a thread
  int mine = 0, loc[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = tid * PER + j;
    loc[j] = mine;
    mine += e < E ? total[e] : 0;
  }
  int inc = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(inc, d, 64);
    if (lane >= d) inc += v;
  }
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int base = inc - mine, valid = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    base += w < wave ? wsum[w] : 0;
    valid += wsum[w];
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = tid * PER + j;
    if (e < E) {
      start[e] += base + loc[j];
      if (b == 0) offsets[e] = base + loc[j];
    }
  }
  if (b == 0 && tid == 0) offsets[E] = valid;
  __syncthreads();

#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const long s = s0 + i * 64;
    if (s < n) {
      int r = -1;
      if (id[i] < E) {
        r = start[id[i]] + wh[wave][id[i]] + rank[i];
        order[r] = (int)s;
      }
      rows[s] = r;
    }
  }
  for (long r = valid + (long)b * T + tid; r < n; r += (long)B * T) order[r] = -1;
}

template <typename Id, int ECAP, int WAVES, int GROUPS>
static void launch_layout(const Id* ids, long n, int E, int* table, int* offsets, int* order, int* rows,
                          hipStream_t stream) {
  constexpr int CH = WAVES * 64 * GROUPS;
  const int B = (int)((n + CH - 1) / CH);
  int bits = 0;
  while ((1 << bits) <= E) ++bits;
  dim3 grid(B < 1 ? 1 : B), block(WAVES * 64);
  if (B <= 1) {
    hipLaunchKernelGGL((layout_place_kernel<Id, ECAP, WAVES, GROUPS, LY_ONE>), grid, block, 0, stream, ids, n, E,
                       bits, table, offsets, order, rows);
    return;
  }
  hipLaunchKernelGGL((layout_count_kernel<Id, CH>), grid, dim3(1024), 0, stream, ids, n, E, table);
  if ((long)B * E <= 65536) {
    hipLaunchKernelGGL((layout_place_kernel<Id, ECAP, WAVES, GROUPS, LY_SUM>), grid, block, 0, stream, ids, n, E,
                       bits, table, offsets, order, rows);
  } else {
    hipLaunchKernelGGL(layout_prefix_kernel, dim3(cdiv(E, 64)), dim3(64), 0, stream, table, B, E);
    hipLaunchKernelGGL((layout_place_kernel<Id, ECAP, WAVES, GROUPS, LY_PREFIX>), grid, block, 0, stream, ids, n,
                       E, bits, table, offsets, order, rows);
  }
}

template <typename Id, int ECAP, int WAVES>
static void layout_sized(const Id* ids, long n, int E, int* table, int* offsets, int* order, int* rows,
                         hipStream_t stream) {
  if (layout_groups(n) == 2) launch_layout<Id, ECAP, WAVES, 2>(ids, n, E, table, offsets, order, rows, stream);
  else launch_layout<Id, ECAP, WAVES, 4>(ids, n, E, table, offsets, order, rows, stream);
}

template <typename Id>
static void layout_any(const Id* ids, long n, int E, int* table, int* offsets, int* order, int* rows,
                       hipStream_t stream) {
  if (E <= 256) layout_sized<Id, 256, 16>(ids, n, E, table, offsets, order, rows, stream);
  else if (E <= 1024) layout_sized<Id, 1024, 16>(ids, n, E, table, offsets, order, rows, stream);
  else layout_sized<Id, 4096, 8>(ids, n, E, table, offsets, order, rows, stream);
}

// whole numbers the table needs: a row a block, and one of sums
extern "C" long lah_ragged_layout_table(long n, int E) {
  const long ch = (E <= 1024 ? 16 : 8) * 64 * layout_groups(n), B = (n + ch - 1) / ch;
  return B <= 1 ? 0 : (B + 1) * E;
}

extern "C" void lah_ragged_layout(const void* ids, int wide, long n, int E, void* table, void* offsets,
                                  void* order, void* rows, hipStream_t stream) {
  if (wide) layout_any((const long*)ids, n, E, (int*)table, (int*)offsets, (int*)order, (int*)rows, stream);
  else layout_any((const int*)ids, n, E, (int*)table, (int*)offsets, (int*)order, (int*)rows, stream);
}
