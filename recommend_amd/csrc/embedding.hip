// Embedding lookup with scaling, out[i] = scale * weight[ids[i]], and its gradient by sorted ids,
//   dW[v] = scale * sum over { i : ids[i] = v } of g[i]        (gfx950).
//
// The gradient never adds with floating atomics.  The ids are sorted together with their positions
// (stable: equal ids keep the order of their positions), so a row's contributions lie side by side;
// lane groups add them in registers in that order and write each row of dW once.  The sums are fp32
// whatever the tensors' type, the same bits on every run, and rounded once.
//
// Up to kFewIds ids one launch does all of it.  Otherwise:
// Sort: up to kRankSortMax ids one launch counts, for every id, the ids that come before it.  More
// ids take an LSD radix sort with digits of up to 9 bits: per digit one launch that counts every
// tile's digits, one that adds up each digit's counts over the tiles and one that places the ids.
// Padded and out-of-range ids get the key `rows`: they come last and add nothing.
//
// Sum: a lane group takes `per_group` consecutive sorted entries and keeps the running row in
// registers.  A row that begins and ends inside the group's entries is written at once; the pieces
// of rows that cross groups are joined in LDS, and the pieces that cross workgroups through memory
// by the closing launch, in the order of the entries.  Rows without an entry are zeroed by further
// workgroups of the same launch, which look their ids up in the sorted keys.
#include <algorithm>

#include "elem.h"

namespace {

// Ids sorted by counting, in one launch whose work grows with their square (whole gradient of 7050 x 64 floats, counting /
// radix sort: 15 / 35 us for 2048 ids, 30 / 41 for 8192, 59 / 43 for 12288).
constexpr int kRankSortMax = 8192;
constexpr int kRankThreads = 16;      // threads that count for one id
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / rk::kWave;
constexpr int kMaxDigitBits = 9;      // one thread for each digit
constexpr int kTileSteps = 8;         // ids of a thread: they stay in registers
constexpr int kTile = kSortThreads * kTileSteps;
// Ids that every summing workgroup sorts itself: one launch instead of three (gradient of 7050 x 64 floats: 3.8 / 6.6 us
// for 16 ids, 7.7 / 10.0 for 256, 11.9 / 11.7 for 512, 17.8 / 12.2 for 640; of 255404 x 128 bf16 14.2 / 19.0 for 512 and
// 20.2 / 19.5 for 640).
constexpr int kFewBits = 9, kFewIds = 1 << kFewBits;
constexpr int32_t kFewRows = 1 << (32 - kFewBits);      // (key and position have to fit a word)
constexpr int kMaxEntries = 1024;     // sorted entries of one workgroup of the summing launch
constexpr int kZeroRows = 256;        // rows that a zeroing workgroup looks up together
// Blocks of them for a workgroup where there are more than the GPU holds at a time (summing launch of 2^20 ids in 30
// million rows of 8 floats: 403 us with four blocks, 579 with one; in 2.2 million rows 53 and 67).
constexpr int kZeroSteps = 4;
constexpr int32_t kManyRows = 2048 * kZeroSteps * kZeroRows;
// Sorted entries of a lane group (whole gradient of 2^20 ids, one of them everywhere, 128 bf16: 207 us with 16, 159 with
// 32, 161 with 64; skewed ids 122 with each; 131072 ids of 1024 floats 210, 191 and 186).
constexpr int kPerGroup = 32;
constexpr int kJoinLanes = 64;       // lanes of a row in the closing launch, at most
// Workgroup borders that one workgroup of the closing launch looks at (8192 ids: 29.6 us with one, 30.0 with four, 31.8
// with 16; 131072 ids of 1024 floats 202, 191 and 191).
constexpr int kJoins = 4;
constexpr int64_t kStreamBytes = 64 << 20;   // looked-up rows from this size on are stored past the caches
// Workgroup pieces of a row above which a whole workgroup joins them (2^20 skewed ids: 130 us with one, 122 with eight,
// 129 with 32; 8192 ids 40, 30 and 30).
constexpr int kLongRun = 8;

// the sort key of an id: ids outside [0, rows) and the padding id go behind all rows
template <typename ID>
__device__ __forceinline__ int32_t key_of(ID id, int32_t rows, int64_t padding) {
  return (id < 0 || (int64_t)id >= rows || (int64_t)id == padding) ? rows : (int32_t)id;
}

// ------------------------------------------------------------------------------------- lookup
// ROWS rows of a lane group are in flight together.  ONCE: the output is larger than what the caches
// should hold and is stored past them; the table's rows stay cached (2^20 rows of 256 bytes from a
// table of 65 MB: 69 us instead of 81, and 20 us less for the launch that follows).
template <typename T, int VEC, typename ID, int ROWS, bool ONCE>
__global__ __launch_bounds__(256) void emb_fwd_kernel(const T *__restrict__ W, int64_t ldw, int32_t rows, int32_t D,
                                                      const ID *__restrict__ ids, int64_t n, float scale, int32_t L,
                                                      T *__restrict__ out) {
  const int G = 256 / L, grp = threadIdx.x / L, l = threadIdx.x - grp * L;
  if (grp >= G) return;
  const int64_t i0 = (int64_t)blockIdx.x * G * ROWS + grp;
  int64_t at[ROWS];
  bool ok[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const ID id = ids[min(i0 + (int64_t)j * G, n - 1)];
    ok[j] = id >= 0 && (int64_t)id < rows;
    at[j] = ok[j] ? (int64_t)id * ldw : 0;
  }
  for (int c0 = l * VEC; c0 < D; c0 += L * VEC) {
    const int col = min(c0, D - VEC);   // the last vector of a row overlaps the one before it
    rk::Pack<T, VEC> v[ROWS];
    if (rows > 0) {
#pragma unroll
      for (int j = 0; j < ROWS; ++j) v[j].load(W + at[j] + col);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
      const int64_t i = i0 + (int64_t)j * G;
      float x[VEC];
      v[j].widen(x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[e] = ok[j] ? x[e] * scale : __builtin_nanf("");   // NaN: no row has this id
      v[j].narrow(x);
      if (i < n) {
        if constexpr (ONCE)
          v[j].store_once(out + i * D + col);
        else
          v[j].store(out + i * D + col);
      }
    }
  }
}

// --------------------------------------------------------------------------------------- sort
// position of id i = number of ids in front of it: smaller keys, and equal keys at lower positions
template <typename ID>
__global__ __launch_bounds__(256) void emb_rank_sort_kernel(const ID *__restrict__ ids, int32_t n, int32_t rows,
                                                            int64_t padding, int32_t *__restrict__ keys,
                                                            int32_t *__restrict__ perm) {
  __shared__ alignas(16) int32_t s_key[kRankSortMax];
  const int32_t room = (n + 3) / 4 * 4;
  for (int j = threadIdx.x; j < room; j += 256) s_key[j] = j < n ? key_of(ids[j], rows, padding) : INT32_MAX;
  __syncthreads();
  const int i = blockIdx.x * (256 / kRankThreads) + threadIdx.x / kRankThreads, sub = threadIdx.x % kRankThreads;
  const int32_t my = i < n ? s_key[i] : 0;
  int before = 0;
#pragma unroll 4
  for (int j = sub * 4; j < room; j += kRankThreads * 4) {
    const int4 k = *reinterpret_cast<const int4 *>(&s_key[j]);
    before += k.x < my + (j < i ? 1 : 0);
    before += k.y < my + (j + 1 < i ? 1 : 0);
    before += k.z < my + (j + 2 < i ? 1 : 0);
    before += k.w < my + (j + 3 < i ? 1 : 0);
  }
#pragma unroll
  for (int off = kRankThreads / 2; off > 0; off >>= 1) before += __shfl_xor(before, off, kRankThreads);
  if (i < n && sub == 0) {
    keys[before] = my;
    perm[before] = i;
  }
}

// source of a radix pass: the ids themselves (first pass) or the keys and positions of the last pass
template <typename ID>
struct FromIds {
  const ID *ids;
  int32_t rows;
  int64_t padding;
  __device__ __forceinline__ int32_t key(int32_t i) const { return key_of(ids[i], rows, padding); }
  __device__ __forceinline__ int32_t pos(int32_t i) const { return i; }
};
struct FromPass {
  const int32_t *keys, *perm;
  __device__ __forceinline__ int32_t key(int32_t i) const { return keys[i]; }
  __device__ __forceinline__ int32_t pos(int32_t i) const { return perm[i]; }
};

template <typename SRC>
__global__ __launch_bounds__(kSortThreads) void emb_count_kernel(SRC src, int32_t n, int shift, int bits,
                                                                 int32_t *__restrict__ counts) {
  __shared__ int32_t s_count[1 << kMaxDigitBits];
  const int nd = 1 << bits;
  if ((int)threadIdx.x < nd) s_count[threadIdx.x] = 0;
  int32_t key[kTileSteps];
  const int64_t lo = (int64_t)blockIdx.x * kTile + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) key[k] = lo + k * kSortThreads < n ? src.key((int32_t)(lo + k * kSortThreads)) : -1;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k)
    if (key[k] >= 0) atomicAdd(&s_count[(key[k] >> shift) & (nd - 1)], 1);
  __syncthreads();
  if ((int)threadIdx.x < nd) counts[(int64_t)blockIdx.x * nd + threadIdx.x] = s_count[threadIdx.x];
}

// exclusive sums of every digit's counts over the tiles, in place, and the digits' totals.  16 digits per
// workgroup (64 bytes of a tile's counts), 16 threads each, which take consecutive shares of the tiles.
__global__ __launch_bounds__(256) void emb_scan_kernel(int32_t *__restrict__ counts, int32_t tiles, int nd,
                                                       int32_t *__restrict__ totals) {
  __shared__ int32_t s_sum[16][16];
  const int q = threadIdx.x / 16, dl = threadIdx.x % 16, d = (int)blockIdx.x * 16 + dl;
  const int32_t share = (tiles + 15) / 16, t0 = min(tiles, q * share), t1 = d < nd ? min(tiles, t0 + share) : t0;
  int32_t sum = 0;
#pragma unroll 8
  for (int32_t t = t0; t < t1; ++t) sum += counts[(int64_t)t * nd + d];
  s_sum[q][dl] = sum;
  __syncthreads();
  int32_t at = 0;
  for (int k = 0; k < q; ++k) at += s_sum[k][dl];
#pragma unroll 8
  for (int32_t t = t0; t < t1; ++t) {
    const int32_t c = counts[(int64_t)t * nd + d];
    counts[(int64_t)t * nd + d] = at;
    at += c;
  }
  if (q == 15 && d < nd) totals[d] = at;
}

// exclusive sum over the threads of a sorting workgroup (s_wave: kSortWaves words of scratch)
__device__ __forceinline__ int32_t block_scan(int32_t v, int32_t *s_wave) {
  const int lane = threadIdx.x % rk::kWave, wave = threadIdx.x / rk::kWave;
  int32_t incl = v;
#pragma unroll
  for (int off = 1; off < rk::kWave; off <<= 1) {
    const int32_t o = __shfl_up(incl, off, rk::kWave);
    if (lane >= off) incl += o;
  }
  if (lane == rk::kWave - 1) s_wave[wave] = incl;
  __syncthreads();
  int32_t at = incl - v;
  for (int w = 0; w < wave; ++w) at += s_wave[w];
  return at;
}

// Places one tile.  Every wavefront owns a consecutive part of it, so that (wavefront, step, lane) is the
// order of the positions and equal digits keep it.  The tile is put in order in LDS first and then
// written from there: ids of one digit go to consecutive places (written straight from the
// registers, 4-byte stores all over the output, this launch took 20 us for 2^20 ids instead of 14).
template <typename SRC>
__global__ __launch_bounds__(kSortThreads) void emb_place_kernel(SRC src, int32_t n, int shift, int bits,
                                                                 const int32_t *__restrict__ counts,
                                                                 const int32_t *__restrict__ totals,
                                                                 int32_t *__restrict__ keys, int32_t *__restrict__ perm) {
  __shared__ int32_t s_off[kSortWaves << kMaxDigitBits];   // [wavefront][digit]: next place in the tile
  __shared__ int32_t s_to[1 << kMaxDigitBits];             // place in the output minus place in the tile
  __shared__ int32_t s_key[kTile], s_pos[kTile];
  __shared__ int32_t s_wave[2][kSortWaves];
  const int nd = 1 << bits, t = threadIdx.x, wave = t / rk::kWave, lane = t % rk::kWave;
  const int64_t tile0 = (int64_t)blockIdx.x * kTile, lo = tile0 + wave * (rk::kWave * kTileSteps) + lane;
  int32_t key[kTileSteps], pos[kTileSteps];
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const bool in = lo + k * rk::kWave < n;
    key[k] = in ? src.key((int32_t)(lo + k * rk::kWave)) : -1;
    pos[k] = in ? src.pos((int32_t)(lo + k * rk::kWave)) : 0;
  }
  const int32_t total = t < nd ? totals[t] : 0, front = t < nd ? counts[(int64_t)blockIdx.x * nd + t] : 0;
  for (int i = t; i < kSortWaves * nd; i += kSortThreads) s_off[i] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k)
    if (key[k] >= 0) atomicAdd(&s_off[wave * nd + ((key[k] >> shift) & (nd - 1))], 1);
  const int32_t out0 = block_scan(total, s_wave[0]) + front;   // (its barrier also closes the counting)
  int32_t mine = 0;
  if (t < nd)
    for (int w = 0; w < kSortWaves; ++w) mine += s_off[w * nd + t];
  int32_t at = block_scan(mine, s_wave[1]);
  if (t < nd) {
    s_to[t] = out0 - at;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t c = s_off[w * nd + t];
      s_off[w * nd + t] = at;
      at += c;
    }
  }
  __syncthreads();
  // rank of a lane among the lanes of its digit, their number and whether it is the last of them: these do
  // not wait for each other, the eight LDS steps below do
  int rank[kTileSteps], same_n[kTileSteps];
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const int d = (key[k] >> shift) & (nd - 1);
    uint64_t same = __ballot(key[k] >= 0);
#pragma unroll
    for (int b = 0; b < kMaxDigitBits; ++b) {            // (bits that a digit does not have are zero in all lanes)
      const bool one = (d >> b) & 1;
      const uint64_t set = __ballot(one);
      same &= one ? set : ~set;
    }
    rank[k] = __popcll(same & ((1ull << lane) - 1));
    same_n[k] = (same >> lane) == 1 ? __popcll(same) : 0;
  }
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    int32_t *off = &s_off[wave * nd + ((key[k] >> shift) & (nd - 1))];
    int32_t first = 0;
    if (key[k] >= 0) {
      first = *off;
      s_key[first + rank[k]] = key[k];
      s_pos[first + rank[k]] = pos[k];
    }
    // (a wavefront's LDS operations complete in program order: all lanes have read before one writes)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (key[k] >= 0 && same_n[k]) *off = first + same_n[k];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  __syncthreads();
  const int count = (int)min((int64_t)kTile, (int64_t)n - tile0);
#pragma unroll
  for (int k = 0; k < kTileSteps; ++k) {
    const int i = k * kSortThreads + t;
    if (i >= count) break;
    const int32_t ky = s_key[i], to = i + s_to[(ky >> shift) & (nd - 1)];
    keys[to] = ky;
    perm[to] = s_pos[i];
  }
}

// ---------------------------------------------------------------------------------------- sum
struct SumArgs {
  const int32_t *keys, *perm;   // sorted ids and where they stood
  int32_t n, rows, D;
  int32_t L, G, per_group;      // lanes of a row, rows side by side in a workgroup, entries of a lane group
  int32_t blocks;               // workgroups that sum; the ones behind them zero
  int32_t zero_steps;           // blocks of kZeroRows rows for each of those, 1 or kZeroSteps
  float scale;
  float *pieces;                // [blocks][2][D]: what a workgroup has of the row it begins / ends in
};

// first place of a key that is not below v
__device__ __forceinline__ int32_t lower_bound(const int32_t *__restrict__ keys, int32_t n, int32_t v) {
  int32_t lo = 0, hi = n;
  while (lo < hi) {
    const int32_t mid = (lo + hi) >> 1;
    if (keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// Zeros in row z * kZeroRows + threadIdx.x where `absent` says so, a wavefront's 64 rows together.  A lane carries row
// and column of its next vector along: the number of the 64 rows' vectors, which rows of 2^25 vectors take past 32 bits,
// is never formed.
template <typename T, int VEC>
__device__ __forceinline__ void zero_rows(int32_t z, bool absent, int32_t D, T *__restrict__ dW) {
  const uint64_t mask = __ballot(absent);
  if (!mask) return;
  const int lane = threadIdx.x % rk::kWave, per_row = (D + VEC - 1) / VEC;
  const int64_t row0 = (int64_t)z * kZeroRows + (threadIdx.x - lane);
  rk::Pack<T, VEC> zero;
#pragma unroll
  for (int i = 0; i < rk::Pack<T, VEC>::kWords; ++i) zero.w[i] = 0u;
  const int step_r = rk::kWave / per_row, step_c = rk::kWave - step_r * per_row;   // (a column step is less than a row)
  int r = lane / per_row, c = lane - r * per_row;
  while (r < rk::kWave) {
    if ((mask >> r) & 1) zero.store(dW + (row0 + r) * D + min(c * VEC, D - VEC));
    r += step_r;
    c += step_c;
    if (c >= per_row) {
      c -= per_row;
      ++r;
    }
  }
}

// The rows of `K` blocks of kZeroRows from block z on: zeros where no sorted key names them.  A thread's K
// searches, chains of loads that wait for each other, run side by side.
template <typename T, int VEC, int K>
__device__ __forceinline__ void zero_absent(const SumArgs &a, int32_t z, T *__restrict__ dW) {
  int32_t v[K], lo[K], len[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = (z + k) * kZeroRows + (int32_t)threadIdx.x;
    lo[k] = 0;
    len[k] = a.n;
  }
  for (int32_t left = a.n; left > 0; left >>= 1) {       // (a step leaves half of `len` at most)
    int32_t key[K];
#pragma unroll
    for (int k = 0; k < K; ++k) key[k] = a.keys[min(lo[k] + (len[k] >> 1), a.n - 1)];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int32_t half = len[k] >> 1;
      const bool up = len[k] > 0 && key[k] < v[k];
      lo[k] = up ? lo[k] + half + 1 : lo[k];
      len[k] = up ? len[k] - half - 1 : half;
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const bool found = lo[k] < a.n && a.keys[min(lo[k], a.n - 1)] == v[k];
    zero_rows<T, VEC>(z + k, v[k] < a.rows && !found, a.D, dW);
  }
}

template <typename T, int VEC>
__device__ __forceinline__ void put_row(T *__restrict__ dst, const float (&acc)[VEC], float scale) {
  float x[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = acc[e] * scale;
  rk::Pack<T, VEC> v;
  v.narrow(x);
  v.store(dst);
}

// Adds a workgroup's `count` sorted entries: key[1 ..] and pos[0 ..], with the key in front of them in key[0]
// and the one behind them in key[1 + count].  pieces: where the parts of rows go that begin in front of
// them or go on behind them (ALONE: none does).
template <typename T, int VEC, bool ALONE>
__device__ __forceinline__ void sum_entries(const SumArgs &a, const T *__restrict__ g, T *__restrict__ dW,
                                            const int32_t *key, const int32_t *pos, int count, int per_group,
                                            float *__restrict__ pieces) {
  constexpr int U = 8;                                   // rows of g in flight per lane group
  __shared__ float s_head[256 * VEC], s_tail[256 * VEC]; // what a group has of the row it begins / ends in
  __shared__ uint8_t s_through[256], s_has_tail[256];
  const int grp = threadIdx.x / a.L, l = threadIdx.x - grp * a.L;
  const int es = min(count, grp * per_group), ee = min(count, es + per_group);
  const bool live = grp < a.G && es < ee;
  const bool began_before = live && key[es] == key[1 + es];

  for (int c0 = 0; c0 < a.D; c0 += a.L * VEC) {
    const bool on = live && c0 + l * VEC < a.D;
    const int col = min(c0 + l * VEC, a.D - VEC), slot = threadIdx.x * VEC;
    bool through = false, has_tail = false;
    if (on) {
      float acc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
      int32_t cur = key[1 + es];
      bool first = began_before;                         // still in the row that an earlier group began
      for (int i = es; i < ee; i += U) {
        rk::Pack<T, VEC> v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) v[j].load_once(g + (int64_t)pos[min(i + j, ee - 1)] * a.D + col);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (i + j >= ee) break;
          const int32_t k = key[1 + i + j];
          if (k != cur) {
            if (first) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) s_head[slot + e] = acc[e];
            } else {
              put_row<T, VEC>(dW + (int64_t)cur * a.D + col, acc, a.scale);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
            cur = k;
            first = false;
          }
          float x[VEC];
          v[j].widen(x);
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += x[e];
        }
      }
      const bool goes_on = key[1 + ee] == cur;
      if (first) {
        through = goes_on;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_head[slot + e] = acc[e];
      } else if (goes_on) {
        has_tail = true;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_tail[slot + e] = acc[e];
      } else {
        put_row<T, VEC>(dW + (int64_t)cur * a.D + col, acc, a.scale);
      }
    }
    if (l == 0 && grp < a.G) {
      s_through[grp] = through;
      s_has_tail[grp] = has_tail;
    }
    __syncthreads();
    if (on && s_has_tail[grp]) {                         // a row begins here and goes on: add the groups behind
      float acc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = s_tail[slot + e];
      int j = grp + 1;
      bool open = true;
      for (; j < a.G && open; ++j) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += s_head[(j * a.L + l) * VEC + e];
        open = s_through[j];
      }
      if (ALONE || !open) {
        put_row<T, VEC>(dW + (int64_t)key[ee] * a.D + col, acc, a.scale);
      } else if constexpr (!ALONE) {
        float *p = pieces + a.D + col;
#pragma unroll
        for (int e = 0; e < VEC; ++e) p[e] = acc[e];
      }
    }
    if (!ALONE && on && grp == 0 && began_before) {      // the row that an earlier workgroup began
      float acc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = s_head[slot + e];
      for (int j = 0; s_through[j] && j + 1 < a.G; ++j) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += s_head[((j + 1) * a.L + l) * VEC + e];
      }
      float *p = pieces + col;
#pragma unroll
      for (int e = 0; e < VEC; ++e) p[e] = acc[e];
    }
    __syncthreads();
  }
}

template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_sum_kernel(SumArgs a, const T *__restrict__ g, T *__restrict__ dW) {
  __shared__ int32_t s_key[kMaxEntries + 2], s_pos[kMaxEntries];
  if ((int32_t)blockIdx.x >= a.blocks) {
    const int32_t z = (int32_t)blockIdx.x - a.blocks;
    if (a.zero_steps == 1)
      zero_absent<T, VEC, 1>(a, z, dW);
    else
      zero_absent<T, VEC, kZeroSteps>(a, z * kZeroSteps, dW);
    return;
  }
  const int per_block = a.G * a.per_group;
  const int32_t s0 = (int32_t)blockIdx.x * per_block, s1 = (int32_t)min((int64_t)a.n, (int64_t)s0 + per_block);
  int count = s1 - s0;
  for (int i = threadIdx.x; i < count; i += 256) {
    s_key[1 + i] = a.keys[s0 + i];
    s_pos[i] = a.perm[s0 + i];
  }
  if (threadIdx.x == 0) {
    s_key[0] = s0 > 0 ? a.keys[s0 - 1] : -1;
    s_key[1 + count] = s1 < a.n ? a.keys[s1] : -1;
  }
  __syncthreads();
  if (s_key[count] >= a.rows) count = lower_bound(s_key + 1, count, a.rows);   // entries that add nothing come last
  if (count == 0) return;
  sum_entries<T, VEC, false>(a, g, dW, s_key, s_pos, count, a.per_group, a.pieces + (int64_t)blockIdx.x * 2 * a.D);
}

// Few ids, one launch: every summing workgroup sorts all of them in LDS, by counting, and takes a share of the
// sorted entries that begins and ends between rows; the zeroing ones look their rows up in the ids.
template <typename T, int VEC, typename ID>
__global__ __launch_bounds__(256) void emb_few_kernel(SumArgs a, const ID *__restrict__ ids, int64_t padding,
                                                      const T *__restrict__ g, T *__restrict__ dW) {
  __shared__ alignas(16) uint32_t s_in[kFewIds];
  __shared__ int32_t s_key[kFewIds + 2], s_pos[kFewIds];
  const int n = a.n;
  if ((int32_t)blockIdx.x >= a.blocks) {
    const int32_t z = (int32_t)blockIdx.x - a.blocks, v = z * kZeroRows + (int32_t)threadIdx.x;
    s_in[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
      const int32_t r = key_of(ids[i], a.rows, padding) - z * kZeroRows;
      if (r >= 0 && r < kZeroRows) s_in[r] = 1;
    }
    __syncthreads();
    zero_rows<T, VEC>(z, v < a.rows && s_in[threadIdx.x] == 0, a.D, dW);
    return;
  }
  // key and position in one word: one comparison orders both
  uint32_t mine[kFewIds / 256];
  int before[kFewIds / 256];
#pragma unroll
  for (int k = 0; k < kFewIds / 256; ++k) {
    const int i = k * 256 + threadIdx.x;
    mine[k] = i < n ? (uint32_t)key_of(ids[i], a.rows, padding) << kFewBits | (uint32_t)i : UINT32_MAX;
    before[k] = 0;
    s_in[i] = mine[k];
  }
  if (threadIdx.x == 0) s_key[0] = s_key[1 + n] = -1;
  __syncthreads();
#pragma unroll 4
  for (int j = 0; j < n; j += 4) {                       // (words behind the last id are larger than all)
    const uint4 c = *reinterpret_cast<const uint4 *>(&s_in[j]);
#pragma unroll
    for (int k = 0; k < kFewIds / 256; ++k)
      before[k] += (c.x < mine[k]) + (c.y < mine[k]) + (c.z < mine[k]) + (c.w < mine[k]);
  }
#pragma unroll
  for (int k = 0; k < kFewIds / 256; ++k)
    if (mine[k] != UINT32_MAX) {
      s_key[1 + before[k]] = (int32_t)(mine[k] >> kFewBits);
      s_pos[before[k]] = (int32_t)(mine[k] & (kFewIds - 1));
    }
  __syncthreads();
  // the share [lo, hi) of this workgroup, moved up to where a row begins
  const int32_t *key = s_key + 1;
  const int valid = lower_bound(key, n, a.rows), share = a.G * a.per_group;
  int lo = min(valid, (int)blockIdx.x * share), hi = min(valid, lo + share);
  if (lo > 0 && lo < valid && key[lo] == key[lo - 1]) lo = lower_bound(key, n, key[lo] + 1);
  if (hi > 0 && hi < valid && key[hi] == key[hi - 1]) hi = lower_bound(key, n, key[hi] + 1);
  if (lo >= hi) return;
  sum_entries<T, VEC, true>(a, g, dW, s_key + lo, s_pos + lo, hi - lo, (hi - lo + a.G - 1) / a.G, a.pieces);
}

// acc += the head pieces of workgroups k0 .. k1, in that order, eight of them in flight
template <int VEC>
__device__ __forceinline__ void add_pieces(const SumArgs &a, int32_t k0, int32_t k1, int col, float (&acc)[VEC]) {
  for (int32_t k = k0; k < k1; k += 8) {
    rk::Pack<float, VEC> v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j].load(a.pieces + (int64_t)min(k + j, k1 - 1) * 2 * a.D + col);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (k + j >= k1) break;
      float x[VEC];
      v[j].widen(x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += x[e];
    }
  }
}

// Rows that cross workgroups: the workgroup in which such a row begins has a tail piece, the ones it
// goes on into have head pieces; they are added in that order.  One lane group per workgroup of the
// summing launch; rows with many pieces are added by the whole workgroup, a consecutive share each.
// Wide rows are cut into slices of kJoinLanes vectors (blockIdx.y), so that enough lane groups share
// the pieces (one id 16384 times, rows of 4000 floats: 50 us instead of 587; slices of 32
// vectors cost ordinary rows of 1024 floats 32 us instead of 20).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void emb_join_kernel(SumArgs a, int32_t L, T *__restrict__ dW) {
  __shared__ float s_part[256 * VEC];
  __shared__ int32_t s_last[kJoins];                       // last workgroup of the row that begins in this one (0: none)
  __shared__ int32_t s_end;
  const int per_block = a.G * a.per_group, G = 256 / L;   // (of the summing launch; lane groups of this one)
  const int grp = threadIdx.x / L, l = threadIdx.x - grp * L;
  const int borders = min(G, kJoins);
  const int32_t b = (int32_t)blockIdx.x * borders + grp;
  int32_t last = 0;
  if (grp < borders && (int64_t)(b + 1) * per_block < a.n) {
    const int32_t s0 = b * per_block, s1 = s0 + per_block, key = a.keys[s1 - 1];
    const bool goes_on = key < a.rows && a.keys[s1] == key;
    const bool began_before = s0 > 0 && a.keys[s0 - 1] == key;
    if (goes_on && !began_before) {
      // how many of the next workgroups begin with the key, eight looked at together
      last = b + 1;
      bool open = true;
      while (open && last - b < kLongRun) {
        int32_t k[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) k[j] = a.keys[(int64_t)min(last + 1 + j, a.blocks - 1) * per_block];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          open = open && last + 1 < a.blocks && k[j] == key;
          last += open ? 1 : 0;
        }
      }
      if (open) last = -1;                               // more than a lane group adds
    }
  }
  if (grp < borders && l == 0) s_last[grp] = last;
  __syncthreads();
  for (int j = 0; j < borders; ++j) {                    // (the same for every thread: barriers inside)
    if (s_last[j] >= 0) continue;
    // the first workgroup that does not begin with the key, 256 looked at together
    const int32_t bj = (int32_t)blockIdx.x * borders + j, key = a.keys[(int64_t)(bj + 1) * per_block - 1];
    if (threadIdx.x == 0) s_end = INT32_MAX;
    __syncthreads();
    for (int32_t k0 = bj + 2;; k0 += 256) {
      const int32_t k = k0 + (int32_t)threadIdx.x;
      if (k >= a.blocks || a.keys[(int64_t)k * per_block] != key) atomicMin(&s_end, k);
      __syncthreads();
      const bool found = s_end != INT32_MAX;
      __syncthreads();                                   // (nobody looks again before everybody has seen it)
      if (found) break;
    }
    if (threadIdx.x == 0) s_last[j] = s_end - 1;
    __syncthreads();
  }
  if (grp < borders) last = s_last[grp];
  for (int64_t c = (int64_t)blockIdx.y * L * VEC; c < a.D; c += (int64_t)gridDim.y * L * VEC) {
    const int c0 = (int)c;
    const bool on = grp < G && c0 + l * VEC < a.D;
    const int col = min(c0 + l * VEC, a.D - VEC);
    if (on && last > 0 && last - b <= kLongRun) {
      float acc[VEC];
      const float *p = a.pieces + ((int64_t)b * 2 + 1) * a.D + col;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = p[e];
      add_pieces<VEC>(a, b + 1, last + 1, col, acc);
      put_row<T, VEC>(dW + (int64_t)a.keys[(int64_t)(b + 1) * per_block - 1] * a.D + col, acc, a.scale);
    }
    for (int j = 0; j < borders; ++j) {                  // (the same for every thread: barriers inside)
      const int32_t bj = (int32_t)blockIdx.x * borders + j, lj = s_last[j], pieces = lj - bj;
      if (lj == 0 || pieces <= kLongRun) continue;
      const int32_t share = (pieces + G - 1) / G;
      if (on) {
        float acc[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
        const int32_t k0 = bj + 1 + grp * share;
        add_pieces<VEC>(a, k0, min(lj + 1, k0 + share), col, acc);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_part[threadIdx.x * VEC + e] = acc[e];
      }
      __syncthreads();
      if (on && grp == 0) {
        float acc[VEC];
        const float *p = a.pieces + ((int64_t)bj * 2 + 1) * a.D + col;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = p[e];
        for (int q = 0; q < G; ++q)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += s_part[(q * L + l) * VEC + e];
        put_row<T, VEC>(dW + (int64_t)a.keys[(int64_t)(bj + 1) * per_block - 1] * a.D + col, acc, a.scale);
      }
      __syncthreads();
    }
  }
}

// --------------------------------------------------------------------------------------- host
struct Layout {              // of the backward workspace, in 4-byte words
  int32_t L, G, per_group, blocks;
  int passes, bits;          // radix passes (0: the ids are sorted by counting) and bits of a digit
  int32_t tiles;
  int64_t keys[2], perm[2], counts, totals, pieces, words;
};

int lanes_of(int32_t D, int32_t dtype) {
  const int full = dtype == RK_F32 ? 4 : 8, vec = D >= full ? full : 1;
  // (four lanes at least: more than 64 rows side by side in a workgroup make long chains of joins)
  return std::max(4, std::min(256, (D + vec - 1) / vec));
}

Layout layout_of(int64_t n, int32_t rows, int32_t D, int32_t dtype) {
  Layout y = {};
  y.L = lanes_of(D, dtype);
  y.G = 256 / y.L;
  // 512 entries for a workgroup where there are enough of them to give every CU some, fewer otherwise
  y.per_group = std::max(4, std::min(kPerGroup, 512 / y.G));
  while (y.per_group > 4 && rk::ceil_div(n, (int64_t)y.G * y.per_group) < 512) y.per_group /= 2;
  y.blocks = (int32_t)rk::ceil_div(n, (int64_t)y.G * y.per_group);
  if (n > kRankSortMax) {
    int key_bits = 1;
    while ((rows >> key_bits) != 0) ++key_bits;          // keys are 0 .. rows
    y.passes = (int)rk::ceil_div(key_bits, kMaxDigitBits);
    y.bits = (int)rk::ceil_div(key_bits, y.passes);
    y.tiles = (int32_t)rk::ceil_div(n, kTile);
  }
  int64_t at = 0;
  const int64_t room = rk::ceil_div(n, 4) * 4;
  for (int k = 0; k < 2; ++k) {
    y.keys[k] = at;
    at += k == 0 || y.passes > 1 ? room : 0;
    y.perm[k] = at;
    at += k == 0 || y.passes > 1 ? room : 0;
  }
  y.counts = at;
  at += (int64_t)y.tiles << y.bits;
  y.totals = at;
  at += 1 << kMaxDigitBits;
  y.pieces = at;
  at += (int64_t)y.blocks * 2 * D;
  y.words = at;
  return y;
}

int check_common(int32_t dtype, int32_t id_bytes, int64_t n, int32_t rows, int32_t D) {
  RK_CHECK_ARG(dtype == RK_F32 || dtype == RK_BF16 || dtype == RK_F16, "unknown element type %d", dtype);
  RK_CHECK_ARG(id_bytes == 4 || id_bytes == 8, "ids are int32 or int64, not of %d bytes", id_bytes);
  RK_CHECK_ARG(n >= 0 && rows >= 0 && D >= 1, "bad size: %lld ids, table %d x %d", (long long)n, rows, D);
  RK_CHECK_ARG(n < (1ll << 31) - (1 << 24) && rows < (1ll << 31) - (1 << 24), "more than 2^31 ids or rows");
  // (a lane's next column is formed before it is compared with the width)
  RK_CHECK_ARG(D < (1ll << 31) - (1 << 24), "more than 2^31 columns");
  return RK_OK;
}

template <typename T, int VEC, typename ID, int ROWS, bool ONCE>
int launch_fwd_as(const void *W, int64_t ldw, int32_t rows, int32_t D, const void *ids, int64_t n, float scale, void *out,
                  int L, hipStream_t st) {
  const int64_t blocks = rk::ceil_div(n, (int64_t)(256 / L) * ROWS);
  RK_CHECK_ARG(blocks < rk::kMaxBlocks256, "too many ids for one call");
  emb_fwd_kernel<T, VEC, ID, ROWS, ONCE><<<(uint32_t)blocks, 256, 0, st>>>((const T *)W, ldw, rows, D, (const ID *)ids, n,
                                                                         scale, L, (T *)out);
  RK_CHECK_LAUNCH("emb_fwd_kernel");
  return RK_OK;
}

template <typename T, int VEC, typename ID>
int launch_fwd(const void *W, int64_t ldw, int32_t rows, int32_t D, const void *ids, int64_t n, float scale, void *out,
               int32_t dtype, hipStream_t st) {
  const int L = lanes_of(D, dtype);
  // two rows per lane group once that still fills the GPU (2^20 rows of 256 bytes: 69 us; one 72, four 72, eight 73)
  if (n < (int64_t)(256 / L) * 2 * 1024)
    return launch_fwd_as<T, VEC, ID, 1, false>(W, ldw, rows, D, ids, n, scale, out, L, st);
  if (n * D * (int64_t)sizeof(T) < kStreamBytes)
    return launch_fwd_as<T, VEC, ID, 2, false>(W, ldw, rows, D, ids, n, scale, out, L, st);
  return launch_fwd_as<T, VEC, ID, 2, true>(W, ldw, rows, D, ids, n, scale, out, L, st);
}

template <typename SRC>
int launch_pass(SRC src, const Layout &y, int32_t n, int pass, int32_t *ws, int to, hipStream_t st) {
  const int shift = pass * y.bits;
  emb_count_kernel<SRC><<<y.tiles, kSortThreads, 0, st>>>(src, n, shift, y.bits, ws + y.counts);
  RK_CHECK_LAUNCH("emb_count_kernel");
  emb_scan_kernel<<<(uint32_t)rk::ceil_div(1 << y.bits, 16), 256, 0, st>>>(ws + y.counts, y.tiles, 1 << y.bits, ws + y.totals);
  RK_CHECK_LAUNCH("emb_scan_kernel");
  emb_place_kernel<SRC><<<y.tiles, kSortThreads, 0, st>>>(src, n, shift, y.bits, ws + y.counts, ws + y.totals,
                                                         ws + y.keys[to], ws + y.perm[to]);
  RK_CHECK_LAUNCH("emb_place_kernel");
  return RK_OK;
}

// the sorted keys and positions end up in buffer 0
template <typename ID>
int launch_sort(const ID *ids, int32_t n, int32_t rows, int64_t padding, const Layout &y, int32_t *ws, hipStream_t st) {
  if (y.passes == 0) {
    emb_rank_sort_kernel<ID><<<(uint32_t)rk::ceil_div(n, 256 / kRankThreads), 256, 0, st>>>(ids, n, rows, padding, ws + y.keys[0],
                                                                           ws + y.perm[0]);
    RK_CHECK_LAUNCH("emb_rank_sort_kernel");
    return RK_OK;
  }
  for (int p = 0; p < y.passes; ++p) {
    const int to = (y.passes - 1 - p) & 1;
    const int rc = p == 0 ? launch_pass(FromIds<ID>{ids, rows, padding}, y, n, p, ws, to, st)
                          : launch_pass(FromPass{ws + y.keys[to ^ 1], ws + y.perm[to ^ 1]}, y, n, p, ws, to, st);
    if (rc) return rc;
  }
  return RK_OK;
}

template <typename T, int VEC, typename ID>
int launch_few(const SumArgs &a, const ID *ids, int64_t padding, const void *g, void *dW, hipStream_t st) {
  const int64_t blocks = (int64_t)a.blocks + rk::ceil_div(a.rows, kZeroRows);
  emb_few_kernel<T, VEC, ID><<<(uint32_t)blocks, 256, 0, st>>>(a, ids, padding, (const T *)g, (T *)dW);
  RK_CHECK_LAUNCH("emb_few_kernel");
  return RK_OK;
}

template <typename T, int VEC>
int launch_sum(const SumArgs &a, const void *g, void *dW, hipStream_t st) {
  const int64_t blocks = (int64_t)a.blocks + rk::ceil_div(a.rows, kZeroRows * a.zero_steps);
  RK_CHECK_ARG(blocks < rk::kMaxBlocks256, "too many ids for one call");
  emb_sum_kernel<T, VEC><<<(uint32_t)blocks, 256, 0, st>>>(a, (const T *)g, (T *)dW);
  RK_CHECK_LAUNCH("emb_sum_kernel");
  if (a.blocks > 1) {
    const int L = std::min(a.L, kJoinLanes);
    const uint32_t slices = (uint32_t)std::min<int64_t>(1024, rk::ceil_div((int64_t)a.D, L * VEC));
    emb_join_kernel<T, VEC><<<dim3((uint32_t)rk::ceil_div(a.blocks - 1, std::min(256 / L, kJoins)), slices), 256, 0, st>>>(a, L, (T *)dW);
    RK_CHECK_LAUNCH("emb_join_kernel");
  }
  return RK_OK;
}

}  // namespace

extern "C" {

int rk_embedding_fwd(const void *weight, int64_t ld_weight, int32_t rows, int32_t D, int32_t dtype, const void *ids,
                     int32_t id_bytes, int64_t n, float scale, void *out, void *stream) {
  if (int rc = check_common(dtype, id_bytes, n, rows, D)) return rc;
  if (n == 0) return RK_OK;
  RK_CHECK_ARG(ids && out && (weight || rows == 0), "null pointer");
  RK_CHECK_ARG(ld_weight >= D || rows <= 1, "rows of the table overlap");
  hipStream_t st = (hipStream_t)stream;
#define RK_FWD(T, VEC)                                                                                       \
  (id_bytes == 8 ? launch_fwd<T, VEC, int64_t>(weight, ld_weight, rows, D, ids, n, scale, out, dtype, st)    \
                 : launch_fwd<T, VEC, int32_t>(weight, ld_weight, rows, D, ids, n, scale, out, dtype, st))
  if (dtype == RK_F32) return D >= 4 ? RK_FWD(float, 4) : RK_FWD(float, 1);
  if (dtype == RK_BF16) return D >= 8 ? RK_FWD(__bf16, 8) : RK_FWD(__bf16, 1);
  return D >= 8 ? RK_FWD(_Float16, 8) : RK_FWD(_Float16, 1);
#undef RK_FWD
}

size_t rk_embedding_bwd_ws_bytes(int64_t n, int32_t rows, int32_t D, int32_t dtype) {
  if (n <= 0 || rows < 0 || D < 1) return 0;
  return (size_t)layout_of(n, rows, D, dtype).words * 4;
}

int rk_embedding_bwd(const void *grad, int32_t dtype, const void *ids, int32_t id_bytes, int64_t n, int32_t rows, int32_t D,
                     float scale, int64_t padding_idx, void *d_weight, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_common(dtype, id_bytes, n, rows, D)) return rc;
  if (rows == 0) return RK_OK;
  RK_CHECK_ARG(d_weight && (n == 0 || (grad && ids && ws)), "null pointer");
  RK_CHECK_ARG(ws_bytes >= rk_embedding_bwd_ws_bytes(n, rows, D, dtype), "workspace too small");
  hipStream_t st = (hipStream_t)stream;
  int32_t *w = (int32_t *)ws;
  const Layout y = layout_of(n, rows, D, dtype);
  if (n > 0 && n <= kFewIds && rows < kFewRows - 1) {
    const SumArgs a = {nullptr, nullptr, (int32_t)n, rows, D, y.L, y.G, y.per_group, y.blocks, 1, scale, (float *)w};
#define RK_FEW(T, VEC)                                                          \
  (id_bytes == 8 ? launch_few<T, VEC>(a, (const int64_t *)ids, padding_idx, grad, d_weight, st) \
                 : launch_few<T, VEC>(a, (const int32_t *)ids, padding_idx, grad, d_weight, st))
    if (dtype == RK_F32) return D >= 4 ? RK_FEW(float, 4) : RK_FEW(float, 1);
    if (dtype == RK_BF16) return D >= 8 ? RK_FEW(__bf16, 8) : RK_FEW(__bf16, 1);
    return D >= 8 ? RK_FEW(_Float16, 8) : RK_FEW(_Float16, 1);
#undef RK_FEW
  }
  if (n > 0) {
    const int rc = id_bytes == 8 ? launch_sort((const int64_t *)ids, (int32_t)n, rows, padding_idx, y, w, st)
                                 : launch_sort((const int32_t *)ids, (int32_t)n, rows, padding_idx, y, w, st);
    if (rc) return rc;
  }
  const SumArgs a = {w + y.keys[0], w + y.perm[0], (int32_t)n, rows, D, y.L, y.G, y.per_group, y.blocks,
                     rows < kManyRows ? 1 : kZeroSteps, scale, (float *)(w + y.pieces)};
  if (dtype == RK_F32) return D >= 4 ? launch_sum<float, 4>(a, grad, d_weight, st) : launch_sum<float, 1>(a, grad, d_weight, st);
  if (dtype == RK_BF16) return D >= 8 ? launch_sum<__bf16, 8>(a, grad, d_weight, st) : launch_sum<__bf16, 1>(a, grad, d_weight, st);
  return D >= 8 ? launch_sum<_Float16, 8>(a, grad, d_weight, st) : launch_sum<_Float16, 1>(a, grad, d_weight, st);
}

}  // extern "C"
