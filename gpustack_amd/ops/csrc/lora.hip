// Low-rank adapters of many requests beside a shared projection, for MI355X (gfx950):
//   out[m, n] += sum_j h[m, p R + j] b[s, n, j],   h[m, c] = sum_k x[m, k] a[s, c, k]
// for every row m whose request has adapter s; p: the part (q, k, v; gate, up) that
// column n belongs to; j below the adapter's own rank, what lies behind it in a and b
// is not used. The rows come in an order in which those of one adapter are neighbours
// (order, starts), so a tile of 16 TT rows has one adapter and the matrix unit's
// 16 x 16 x 32 products serve decode steps and prompts alike.
//
// Two launches. The first multiplies by a, with k cut over the grid and over a
// workgroup's four waves: a wave's rows and weights go straight to its registers,
// each read once. Its fp32 sums (h, in `splits` parts) are added up by the second,
// which holds them as two bf16 parts (the value and what that rounded away, 16 bits of
// it in all): one would cost h the 2^-9 that the rest of the sum does not lose. Both
// are bound by memory: x and a, then b and out.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) short s16x8;

DEVICE_INLINE f32x4 multiply(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(s16x8, a),
                                                 __builtin_bit_cast(s16x8, b), c, 0, 0, 0);
}

struct Place { int slot, first, count, rank; };

// Tile `tile` of the list that has ceil(rows / ROWS) of each slot: count 0 where there
// is none. All lanes of all waves agree. Offsets are held within the order's length.
template <int ROWS>
DEVICE_INLINE Place find_tile(int tile, const int* starts, const int* ranks, int S, int T,
                              int R) {
  const int lane = threadIdx.x & (WAVE_SIZE - 1);
  int before = 0;
  for (int s0 = 0; s0 < S; s0 += WAVE_SIZE) {
    const int s = s0 + lane;
    int from = 0, count = 0, rank = 0;
    if (s < S) {
      from = min(max(starts[s], 0), T);
      count = max(min(starts[s + 1], T) - from, 0);
      rank = min(max(ranks[s], 0), R);
    }
    const int mine = (count + ROWS - 1) / ROWS;
    int sum = mine;                          // tiles up to this slot
#pragma unroll
    for (int d = 1; d < WAVE_SIZE; d *= 2) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const unsigned long found = __ballot(before + sum > tile);
    if (found) {
      const int at = __ffsll((unsigned long long)found) - 1;
      const int k = tile - before - __shfl(sum - mine, at);
      const int first = __shfl(from, at) + k * ROWS;
      auto one = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
      return Place{one(s0 + at), one(first),
                   one(min(ROWS, __shfl(from + count, at) - first)),
                   one(__shfl(rank, at))};
    }
    before += __shfl(sum, WAVE_SIZE - 1);
  }
  return Place{0, 0, 0, 0};
}

// h, [splits, T, C] by place in the order. Tiles of 16 TT rows; CT tiles of 16 of the
// C = P R columns, of which an adapter has the ceil(rank / 16) first of each part.
template <int TT, int CT>
__global__ __launch_bounds__(256) void lora_down_kernel(
    float* __restrict__ h, const unsigned short* __restrict__ x, long xs,
    const unsigned short* __restrict__ a, const int* __restrict__ order,
    const int* __restrict__ starts, const int* __restrict__ ranks, int rows, int T, int S,
    int K, int P, int R) {
  constexpr int ROWS = 16 * TT, U = 64;
  __shared__ f32x4 red[4 * TT * CT * WAVE_SIZE];
  const Place p = find_tile<ROWS>(blockIdx.x, starts, ranks, S, T, R);
  const int each = (p.rank + 15) / 16;       // tiles of a part
  const int c0 = blockIdx.y * CT;
  if (p.count == 0 || c0 >= P * each) return;
  const int tid = threadIdx.x, lane = tid & (WAVE_SIZE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE_SIZE);
  const int lc = lane & 15, lg = lane >> 4;
  const int C = P * R;

  const unsigned short* xp[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int row = order[p.first + min(t * 16 + lc, p.count - 1)];
    xp[t] = x + min(max(row, 0), rows - 1) * xs + lg * 16;
  }
  const unsigned short* ap[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) {
    const int i = min(c0 + c, P * each - 1);
    const int j = min(i % each * 16 + lc, p.rank - 1);
    ap[c] = a + ((long)p.slot * C + i / each * R + j) * K + lg * 16;
  }
  const int units = (K + U - 1) / U, splits = gridDim.z;
  const int from = (int)((long)units * blockIdx.z / splits);
  const int to = (int)((long)units * (blockIdx.z + 1) / splits);
  f32x4 acc[TT][CT];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};

  // a lane's 16 neighbours of a unit of 64 k, 8 for each of two products
  for (int u = from + wave; u < to; u += 4) {
    const int k = u * U;
    u32x4 fx[TT][2], fa[CT][2];
    auto piece = [&](const unsigned short* q, int i) {
      const bool in = k + lg * 16 + i * 8 < K;
      u32x4 v = *reinterpret_cast<const u32x4*>(in ? q + k + i * 8 : q - lg * 16);
      if (!in) v = u32x4{0, 0, 0, 0};
      return v;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int t = 0; t < TT; ++t) fx[t][i] = piece(xp[t], i);
#pragma unroll
      for (int c = 0; c < CT; ++c) fa[c][i] = piece(ap[c], i);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int c = 0; c < CT; ++c)
          acc[t][c] = multiply(fa[c][i], fx[t][i], acc[t][c]);
  }
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int c = 0; c < CT; ++c)
      red[((wave * TT + t) * CT + c) * WAVE_SIZE + lane] = acc[t][c];
  __syncthreads();
  // D[column = lg * 4 + r][row = lc] per tile
  for (int i = wave; i < TT * CT; i += 4) {
    f32x4 v = red[i * WAVE_SIZE + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += red[(w * TT * CT + i) * WAVE_SIZE + lane];
    const int row = i / CT * 16 + lc, c = c0 + i % CT;
    const int j = c % each * 16 + lg * 4;
    if (row < p.count && c < P * each && j < R)
      *reinterpret_cast<f32x4*>(h + ((long)blockIdx.z * T + p.first + row) * C +
                                c / each * R + j) = v;
  }
}

struct Ends { int n, end[4]; };

// out += h b^T. A workgroup has 16 TT rows and 256 columns of one part, its waves 64
// each: four tiles of 16 weight rows, dealt so that a lane ends with 16 neighbours of
// a row. KT: 32 k of the rank at a time that the registers hold (32 KT >= rank).
template <int TT, int KT>
__global__ __launch_bounds__(256) void lora_up_kernel(
    unsigned short* __restrict__ out, long os, const float* __restrict__ h, int splits,
    const unsigned short* __restrict__ b, const int* __restrict__ order,
    const int* __restrict__ starts, const int* __restrict__ ranks, int rows, int T, int S,
    int N, int R, Ends ends) {
  constexpr int ROWS = 16 * TT, LD = 32 * KT + 8;
  __shared__ __attribute__((aligned(16))) unsigned short part[2][ROWS * LD];
  const Place p = find_tile<ROWS>(blockIdx.x, starts, ranks, S, T, R);
  if (p.count == 0 || p.rank == 0) return;
  const int tid = threadIdx.x, lane = tid & (WAVE_SIZE - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE_SIZE);
  const int lc = lane & 15, lg = lane >> 4;
  const int C = ends.n * R;

  int block = blockIdx.y, which = 0, low = 0, high = ends.end[0];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int blocks = (high - low + 255) / 256;
    if (i < ends.n - 1 && which == i && block >= blocks) {
      block -= blocks;
      which = i + 1;
      low = high;
      high = ends.end[i + 1];
    }
  }
  const int n0 = low + block * 256 + wave * 64;

  for (int i = tid; i < ROWS * 8 * KT; i += 256) {
    const int row = i / (8 * KT), j = i % (8 * KT) * 4;
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (row < p.count && j < p.rank) {
      const float* at = h + (long)(p.first + row) * C + which * R + j;
      for (int s = 0; s < splits; ++s)
        v += *reinterpret_cast<const f32x4*>(at + (long)s * T * C);
    }
    u16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (j + e >= p.rank) v[e] = 0.f;
      hi[e] = f2bf(v[e]);
      lo[e] = f2bf(v[e] - bf2f(hi[e]));
    }
    *reinterpret_cast<u16x4*>(&part[0][row * LD + j]) = hi;
    *reinterpret_cast<u16x4*>(&part[1][row * LD + j]) = lo;
  }
  __syncthreads();
  if (n0 >= high) return;

  f32x4 acc[TT][4];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[t][c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    if (k * 32 >= p.rank) break;
    const int j = k * 32 + lg * 8, left = p.rank - j;
    u32x4 fb[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      // row i of tile c is column i / 4 * 16 + c * 4 + i % 4
      const int col = min(n0 + (lc >> 2) * 16 + c * 4 + (lc & 3), high - 1);
      fb[c] = u32x4{0, 0, 0, 0};
      if (left > 0) {
        fb[c] = *reinterpret_cast<const u32x4*>(b + ((long)p.slot * N + col) * R + j);
        if (left < 8)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            fb[c][e] &= 2 * e + 1 < left ? ~0u : 2 * e < left ? 0xffffu : 0u;
      }
    }
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const u32x4 hi = *reinterpret_cast<const u32x4*>(&part[0][(t * 16 + lc) * LD + j]);
      const u32x4 lo = *reinterpret_cast<const u32x4*>(&part[1][(t * 16 + lc) * LD + j]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        acc[t][c] = multiply(fb[c], lo, multiply(fb[c], hi, acc[t][c]));
    }
  }
  // acc[t][c][r]: row t * 16 + lc, column lg * 16 + c * 4 + r; ends are multiples of 8
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int i = t * 16 + lc;
    if (i >= p.count) continue;
    const int row = order[p.first + i];
    if (row < 0 || row >= rows) continue;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int col = n0 + lg * 16 + g * 8;
      if (col >= high) continue;
      u16x8* at = reinterpret_cast<u16x8*>(out + row * os + col);
      const u16x8 old = *at;
      u16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = f2bf(bf2f(old[e]) + acc[t][g * 2 + e / 4][e % 4]);
      *at = v;
    }
  }
}

}  // namespace

int lora_most_rank() { return 256; }

// rows: of x and out; T: entries of the order. K, R and the ends are multiples of 8.
// tt (1 or 4): tiles of 16 rows a workgroup.
void lora_launch(void* out, long os, float* h, const void* x, long xs, const void* a,
                 const void* b, const int* order, const int* starts, const int* ranks,
                 int rows, int T, int S, int N, int K, int P, const int* ends, int R,
                 int tt, int splits, hipStream_t s) {
  const int each = 16 * tt;
  // of S slots at most T have rows
  const int tiles = (int)min((long)T, (T + (long)min(S, T) * (each - 1)) / each);
  const int groups = P * ((R + 15) / 16);
  auto down = [&](auto kernel, int ct) {
    hipLaunchKernelGGL(kernel, dim3(tiles, (groups + ct - 1) / ct, splits), dim3(256), 0,
                       s, h, (const unsigned short*)x, xs, (const unsigned short*)a,
                       order, starts, ranks, rows, T, S, K, P, R);
  };
  if (tt == 1) down(lora_down_kernel<1, 1>, 1);
  else down(lora_down_kernel<4, 4>, 4);
  Ends e{P, {0, 0, 0, 0}};
  int blocks = 0;
  for (int i = 0; i < P; ++i) {
    e.end[i] = ends[i];
    blocks += (ends[i] - (i ? ends[i - 1] : 0) + 255) / 256;
  }
  auto up = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(tiles, blocks), dim3(256), 0, s,
                       (unsigned short*)out, os, h, splits, (const unsigned short*)b,
                       order, starts, ranks, rows, T, S, N, R, e);
  };
  if (tt == 1) {
    if (R <= 32) up(lora_up_kernel<1, 1>);
    else if (R <= 64) up(lora_up_kernel<1, 2>);
    else if (R <= 128) up(lora_up_kernel<1, 4>);
    else up(lora_up_kernel<1, 8>);
  } else {
    if (R <= 32) up(lora_up_kernel<4, 1>);
    else if (R <= 64) up(lora_up_kernel<4, 2>);
    else if (R <= 128) up(lora_up_kernel<4, 4>);
    else up(lora_up_kernel<4, 8>);
  }
}
