// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// Lookup: out[i] = scale * table[tok[i]].  Each row is read and written once,
// in 16-byte pieces where the rows are aligned; memory is the bound: 524,288
// rows of 512 bytes from 262,144 take 102 us, 4.0 TB/s where a large copy
// reaches 4.8.
//
// Gradient: dtable[v] = scale * sum of dout[i] over tok[i] = v.  The tokens
// are sorted with their positions (stable, so a row's positions are in
// order), start[v] is found at the sorted tokens' boundaries, and each table
// row's terms (at most kLong) are added in float32, in that order, by the lanes
// that hold its columns, and the row is written once: no atomics on values, the
// same bits every time, and rows without a token cost their zeros.  A crowded
// row (more terms: grid cells near an object) is cut into pieces of kPiece
// terms, a wave each, whose sums (in float64: the terms may be many) are added
// in order by a last pass.  Where pieces lie in the workspace is decided by an atomic counter; no
// sum depends on it.  524,288 tokens, 262,144 rows of 512 bytes: the sort 53 us,
// the starts 5, the rows 142 (2.8 TB/s: scattered rows behind two dependent
// loads), the crowded rows 23.  16,384 tokens, 8,192 rows of 383 float32: the
// sort 13 us, the rows 18, the crowded rows 12.
#include "nsfps_launch.h"
#include "nsfps_seq_device.h"

#include <algorithm>
#include <type_traits>

#pragma clang fp contract(fast)

namespace nsfps {

using namespace seq;

namespace {

constexpr uint32_t kLong = 16;   // terms that a row adds by itself
constexpr uint32_t kPiece = 64;  // terms of a piece of a longer one

// Workgroups of a grid-stride kernel: a launch holds fewer than 2^32 threads.
uint32_t grid_of(uint64_t blocks) { return (uint32_t)std::min<uint64_t>(blocks, 1u << 20); }

// ---- lookup

// tpr threads (a power of two, at most 256) per row, V elements each
template <typename T, int V>
__global__ __launch_bounds__(256) void k_embed(const T *__restrict__ table,
                                               const int32_t *__restrict__ tokens,
                                               T *__restrict__ out, uint32_t count, uint32_t rows,
                                               uint32_t vecs, uint64_t table_stride,
                                               uint64_t out_stride, float scale, uint32_t tpr) {
  const uint32_t per = 256 / tpr;
  for (uint64_t i = (uint64_t)blockIdx.x * per + threadIdx.x / tpr; i < count;
       i += (uint64_t)gridDim.x * per) {
    const int32_t tok = tokens[i];
    const bool hit = tok >= 0 && (uint32_t)tok < rows;
    const T *src = table + (hit ? (uint64_t)tok * table_stride : 0);
    T *dst = out + i * out_stride;
    for (uint32_t c = threadIdx.x % tpr; c < vecs; c += tpr) {
      float v[V];
      if (hit) {
        load_f32<T, V>(src + (uint64_t)c * V, v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = 0.f;
      }
      store_f32<T, V>(dst + (uint64_t)c * V, v);
    }
  }
}

// ---- gradient

// Stable radix sort of the tokens with their positions, up to kDigitBits bits
// a pass, so that a vocabulary of 2^20 rows takes two.  A pass: each
// workgroup's digit counts (hist[tile][digit]); their sums over the tiles
// ahead, and the digits' totals; the scatter.  A workgroup's kTokTile tokens
// are four waves' runs of 512 in order; a wave ranks 64 at a time by ballots.
// (The sampling build's 8-bit sort of 4,096-key tiles took 99 us for 524,288
// tokens of 19 bits, this one 39; for 16,384 tokens of 14 bits one workgroup
// in LDS took 34 us, one pass over whole keys takes 13.)
constexpr int kDigitBits = 10;
constexpr uint32_t kTokTile = 2048;
constexpr int kTokRounds = kTokTile / 256;

// A token's sort key: itself, or rows when it is outside.
__device__ __forceinline__ uint32_t token_key(const int32_t *tokens, const uint32_t *keys,
                                              uint32_t i, uint32_t rows) {
  if (keys) return keys[i];
  const int32_t t = tokens[i];
  return t >= 0 && (uint32_t)t < rows ? (uint32_t)t : rows;
}

// keys null: the first pass, from the tokens; it clears the counters too.
// A key's digit, (key >> shift) & mask, is below digits.
template <uint32_t kThreads, uint32_t kTile>
__global__ __launch_bounds__(kThreads) void k_token_hist(
    const int32_t *__restrict__ tokens, const uint32_t *__restrict__ keys, uint32_t count,
    uint32_t rows, int shift, uint32_t digits, uint32_t mask, uint32_t *__restrict__ hist,
    uint32_t *__restrict__ counters) {
  constexpr uint32_t kRounds = kTile / kThreads;
  extern __shared__ uint32_t s_cnt[];
  if (!keys && blockIdx.x == 0 && threadIdx.x < 2) counters[threadIdx.x] = 0;
  for (uint32_t d = threadIdx.x; d < digits; d += kThreads) s_cnt[d] = 0;
  __syncthreads();
  const uint64_t base = (uint64_t)blockIdx.x * kTile;
  uint32_t key[kRounds];
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r) {
    const uint64_t i = base + r * kThreads + threadIdx.x;
    key[r] = i < count ? token_key(tokens, keys, (uint32_t)i, rows) : 0u;
  }
#pragma unroll
  for (uint32_t r = 0; r < kRounds; ++r)
    if (base + r * kThreads + threadIdx.x < count)
      atomicAdd(&s_cnt[(key[r] >> shift) & mask], 1u);
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < digits; d += kThreads)
    hist[(uint64_t)blockIdx.x * digits + d] = s_cnt[d];
}

// hist[tile][digit] becomes the digit's count in the tiles ahead; totals[digit].
// 64 digits a workgroup, its 16 waves a run of the tiles each.
__global__ __launch_bounds__(1024) void k_token_scan(uint32_t *__restrict__ hist, uint32_t tiles,
                                                     uint32_t digits,
                                                     uint32_t *__restrict__ totals) {
  __shared__ uint32_t s_sum[16][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t d = blockIdx.x * 64 + lane, run = ceil_div(tiles, 16);
  const uint32_t a = min(wave * run, tiles), b = min(a + run, tiles);
  constexpr uint32_t kAhead = 8;
  uint32_t sum = 0;
  if (d < digits)
    for (uint32_t t = a; t < b; t += kAhead) {
      uint32_t v[kAhead];
#pragma unroll
      for (uint32_t k = 0; k < kAhead; ++k)
        v[k] = t + k < b ? hist[(uint64_t)(t + k) * digits + d] : 0u;
#pragma unroll
      for (uint32_t k = 0; k < kAhead; ++k) sum += v[k];
    }
  s_sum[wave][lane] = sum;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < 16; ++w) {
    before += w < wave ? s_sum[w][lane] : 0u;
    all += s_sum[w][lane];
  }
  if (d >= digits) return;
  if (wave == 0) totals[d] = all;
  for (uint32_t t = a; t < b; t += kAhead) {
    uint32_t v[kAhead];
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k)
      v[k] = t + k < b ? hist[(uint64_t)(t + k) * digits + d] : 0u;
#pragma unroll
    for (uint32_t k = 0; k < kAhead; ++k) {
      if (t + k < b) hist[(uint64_t)(t + k) * digits + d] = before;
      before += v[k];
    }
  }
}

__global__ __launch_bounds__(256) void k_token_scatter(
    const int32_t *__restrict__ tokens, const uint32_t *__restrict__ kin,
    const uint32_t *__restrict__ vin, uint32_t *__restrict__ kout, uint32_t *__restrict__ vout,
    uint32_t count, uint32_t rows, int shift, int bits, const uint32_t *__restrict__ hist,
    const uint32_t *__restrict__ totals) {
  __shared__ uint32_t s_cnt[4][1 << kDigitBits];  // per wave, then the digits' first places
  __shared__ uint32_t s_wave[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, digits = 1u << bits;
  const uint64_t lt = lane ? (~0ull >> (64 - lane)) : 0ull;
  const uint64_t base = (uint64_t)blockIdx.x * kTokTile + wave * (kTokTile / 4);
  uint32_t key[kTokRounds], val[kTokRounds], rank[kTokRounds];
#pragma unroll
  for (int r = 0; r < kTokRounds; ++r) {
    const uint64_t i = base + r * 64 + lane;
    key[r] = i < count ? token_key(tokens, kin, (uint32_t)i, rows) : 0u;
    val[r] = i < count ? (kin ? vin[i] : (uint32_t)i) : 0u;
  }
  // this thread's digits, 4 tid .. 4 tid + 3: their places in the whole order
  uint32_t tot[4], first[4];
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t d = 4 * tid + k;
    tot[k] = d < digits ? totals[d] : 0u;
    first[k] = d < digits ? hist[(uint64_t)blockIdx.x * digits + d] : 0u;
  }
  for (uint32_t d = tid; d < 4 * digits; d += 256) s_cnt[d / digits][d % digits] = 0;
  uint32_t sum = tot[0] + tot[1] + tot[2] + tot[3];
  const uint32_t own = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(sum, off, 64);
    if (lane >= (uint32_t)off) sum += o;
  }
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  sum -= own;
  for (uint32_t w = 0; w < wave; ++w) sum += s_wave[w];
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    first[k] += sum;
    sum += tot[k];
  }
#pragma unroll
  for (int r = 0; r < kTokRounds; ++r) {
    const bool valid = base + r * 64 + lane < count;
    const uint32_t d = (key[r] >> shift) & (digits - 1);
    uint64_t peers = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot((d >> b) & 1u);
      peers &= ((d >> b) & 1u) ? m : ~m;
    }
    const uint32_t before = (uint32_t)__popcll(peers & lt);
    const uint32_t baseq = valid ? s_cnt[wave][d] : 0u;
    rank[r] = baseq + before;
    // all lanes read their base before a leader writes (in-order LDS, one wave)
    __builtin_amdgcn_s_waitcnt(0xc07f);
    if (valid && before == 0) s_cnt[wave][d] = baseq + (uint32_t)__popcll(peers);
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
  __syncthreads();
#pragma unroll
  for (uint32_t k = 0; k < 4; ++k) {
    const uint32_t d = 4 * tid + k;
    if (d >= digits) continue;
    uint32_t at = first[k];
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const uint32_t n = s_cnt[w][d];
      s_cnt[w][d] = at;
      at += n;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTokRounds; ++r) {
    if (base + r * 64 + lane >= count) continue;
    const uint32_t at = s_cnt[wave][(key[r] >> shift) & (digits - 1)] + rank[r];
    kout[at] = key[r];
    vout[at] = val[r];
  }
}

// The scatter of a sort in one pass, a digit being a whole key (0 .. rows): the
// digits' first places are start itself.  Eight waves rank 128 tokens each, so
// that a wave's count of a key fits a byte.
constexpr uint32_t kPlaceTile = 1024, kPlaceThreads = 512, kPlaceWaves = 8;
constexpr uint32_t kPlaceDigits = 12288;  // what 160 KB of LDS hold
constexpr int kPlaceQuads = kPlaceDigits / 4 / kPlaceThreads;
constexpr uint32_t place_lds(uint32_t digits) { return ((digits + 3) & ~3u) * (4 + kPlaceWaves); }

__global__ __launch_bounds__(512) void k_token_place(const int32_t *__restrict__ tokens,
                                                     uint32_t *__restrict__ pos, uint32_t count,
                                                     uint32_t rows, int bits,
                                                     const uint32_t *__restrict__ hist,
                                                     const uint32_t *__restrict__ totals,
                                                     uint32_t *__restrict__ start) {
  // first places [d4], then the waves' counts [waves][d4]
  extern __shared__ __attribute__((aligned(16))) uint32_t s_first[];
  __shared__ uint32_t s_wave[kPlaceWaves];
  constexpr int kRounds = kPlaceTile / kPlaceThreads;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, digits = rows + 1,
                 d4 = (digits + 3) & ~3u, quads = d4 / 4, each = ceil_div(quads, kPlaceThreads);
  uint8_t *const s_cnt = (uint8_t *)(s_first + d4);
  const uint64_t lt = lane ? (~0ull >> (64 - lane)) : 0ull;
  const uint64_t base = (uint64_t)blockIdx.x * kPlaceTile + wave * (kPlaceTile / kPlaceWaves);
  uint32_t key[kRounds], at[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint64_t i = base + r * 64 + lane;
    key[r] = i < count ? token_key(tokens, nullptr, (uint32_t)i, rows) : 0u;
  }
  // this thread's digits: `each` (at most kPlaceQuads) quads of them, one after another.
  // Past the last digit the arrays' padding is read and written; no sum that
  // is used has it.
  uint4 q[kPlaceQuads];
#pragma unroll
  for (int k = 0; k < kPlaceQuads; ++k) {
    const uint32_t v = tid * each + k;
    q[k] = (uint32_t)k < each && v < quads ? ((const uint4 *)totals)[v] : make_uint4(0, 0, 0, 0);
  }
  for (uint32_t v = tid; v < quads * kPlaceWaves / 4; v += kPlaceThreads)
    ((uint4 *)s_cnt)[v] = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) at[r] = hist[(uint64_t)blockIdx.x * digits + key[r]];
  uint32_t sum = 0;
#pragma unroll
  for (int k = 0; k < kPlaceQuads; ++k) sum += q[k].x + q[k].y + q[k].z + q[k].w;
  const uint32_t own = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t o = __shfl_up(sum, off, 64);
    if (lane >= (uint32_t)off) sum += o;
  }
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  sum -= own;
#pragma unroll
  for (uint32_t w = 0; w < kPlaceWaves; ++w) sum += w < wave ? s_wave[w] : 0u;
#pragma unroll
  for (int k = 0; k < kPlaceQuads; ++k) {
    const uint32_t v = tid * each + k;
    if ((uint32_t)k >= each || v >= quads) continue;
    const uint4 f = make_uint4(sum, sum + q[k].x, sum + q[k].x + q[k].y,
                               sum + q[k].x + q[k].y + q[k].z);
    sum = f.w + q[k].w;
    ((uint4 *)s_first)[v] = f;
    if (blockIdx.x == 0) ((uint4 *)start)[v] = f;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool valid = base + r * 64 + lane < count;
    const uint32_t d = key[r];
    uint64_t peers = __ballot(valid);
    for (int k = 0; k < bits; ++k) {
      const uint64_t m = __ballot((d >> k) & 1u);
      peers &= ((d >> k) & 1u) ? m : ~m;
    }
    const uint32_t before = (uint32_t)__popcll(peers & lt);
    const uint32_t baseq = valid ? s_cnt[wave * d4 + d] : 0u;
    at[r] += baseq + before;
    // all lanes read their base before a leader writes (in-order LDS, one wave)
    __builtin_amdgcn_s_waitcnt(0xc07f);
    if (valid && before == 0)
      s_cnt[wave * d4 + d] = (uint8_t)(baseq + (uint32_t)__popcll(peers));
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint64_t i = base + r * 64 + lane;
    if (i >= count) continue;
    uint32_t place = s_first[key[r]] + at[r];
#pragma unroll
    for (uint32_t w = 0; w < kPlaceWaves; ++w) place += w < wave ? s_cnt[w * d4 + key[r]] : 0u;
    pos[place] = (uint32_t)i;
  }
}

// At most 512 tokens: a token's place is the number of tokens before it, those
// of a smaller key and those of its own that come first.  A table too large for
// one pass costs six launches else (us a gradient with them and with this one,
// bf16: 3 tokens of 39,481 rows of 58 32, 14; 395 56, 51; 512 55, 54; 576 55.5,
// 56; 1,024 52, 70; 512 tokens of 262,144 rows of 256 93, 89; 640 90, 90).
constexpr uint32_t kRankTokens = 512;
__global__ __launch_bounds__(kRankTokens) void k_token_rank(const int32_t *__restrict__ tokens,
                                                     uint32_t *__restrict__ kout,
                                                     uint32_t *__restrict__ vout, uint32_t count,
                                                     uint32_t rows,
                                                     uint32_t *__restrict__ counters) {
  __shared__ __attribute__((aligned(16))) uint32_t s_key[kRankTokens];
  const uint32_t i = threadIdx.x;
  const uint32_t key = i < count ? token_key(tokens, nullptr, i, rows) : ~0u;
  s_key[i] = key;  // past the last token: above every key, as rows is below 2^31
  if (i < 2) counters[i] = 0;
  __syncthreads();
  uint32_t at = 0;
  for (uint32_t j = 0; j < count; j += 4) {
    const uint4 q = *(const uint4 *)(s_key + j);
    at += q.x < key || (q.x == key && j < i);
    at += q.y < key || (q.y == key && j + 1 < i);
    at += q.z < key || (q.z == key && j + 2 < i);
    at += q.w < key || (q.w == key && j + 3 < i);
  }
  if (i >= count) return;
  kout[at] = key;
  vout[at] = i;
}

// start[v] (v <= rows): sorted positions below it hold tokens below v.
// Position p = 0 .. count fills start over (key[p - 1], key[p]], key[-1] = -1
// and key[count] = rows; long gaps are filled by the whole workgroup.
__global__ __launch_bounds__(256) void k_embed_starts(const uint32_t *__restrict__ keys,
                                                      uint32_t count, uint32_t rows,
                                                      uint32_t *__restrict__ start) {
  __shared__ uint32_t s_n, s_lo[256], s_hi[256], s_p[256];
  if (threadIdx.x == 0) s_n = 0;
  __syncthreads();
  const uint64_t p = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (p <= count) {
    const uint32_t lo = p == 0 ? 0u : keys[p - 1] + 1, hi = p == count ? rows : keys[p];
    // entries lo .. hi (none where the token is the one before it, or both are outside)
    if (lo <= hi) {
      if (hi - lo < 16) {
        for (uint32_t v = lo; v <= hi; ++v) start[v] = (uint32_t)p;
      } else {
        const uint32_t k = atomicAdd(&s_n, 1u);
        s_lo[k] = lo;
        s_hi[k] = hi;
        s_p[k] = (uint32_t)p;
      }
    }
  }
  __syncthreads();
  const uint32_t n = s_n;
  for (uint32_t k = 0; k < n; ++k)
    for (uint64_t v = (uint64_t)s_lo[k] + threadIdx.x; v <= s_hi[k]; v += 256) start[v] = s_p[k];
}

// acc += the terms pos[from .. to) of one column vector, in order
template <typename T, int V>
__device__ __forceinline__ void add_terms(const T *__restrict__ dout, uint64_t stride,
                                          const uint32_t *__restrict__ pos, uint32_t from,
                                          uint32_t to, double (&acc)[V]) {
  constexpr uint32_t kAhead = 8;  // loads in flight
  uint32_t p = from;
  for (; p + kAhead <= to; p += kAhead) {
    float v[kAhead][V];
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
      load_f32<T, V>(dout + (uint64_t)pos[p + j] * stride, v[j]);
#pragma unroll
    for (uint32_t j = 0; j < kAhead; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += v[j][k];
  }
  for (; p < to; ++p) {
    float v[V];
    load_f32<T, V>(dout + (uint64_t)pos[p] * stride, v);
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += v[k];
  }
}

struct LongRow {
  uint32_t row, piece;  // the row, and its first piece in the workspace
};

// Table rows, `lpr` lanes (a power of two, at most 256) a row.  Most rows have
// few terms, so what a row costs is a chain of dependent loads (its start, its
// positions, its terms): a lane group takes kRows rows at a time, kTerms terms
// of each a round, and issues each link of their chains together.  Crowded
// rows are listed: counters[0] counts them, counters[1] their pieces;
// piece_at[k] = the sorted positions of piece k.
template <typename T, typename G, int V>
__global__ __launch_bounds__(256) void k_embed_rows(
    const T *__restrict__ dout, uint64_t dout_stride, const uint32_t *__restrict__ pos,
    const uint32_t *__restrict__ start, G *__restrict__ dtable, uint64_t table_stride,
    uint32_t rows, uint32_t vecs, uint32_t lpr, float scale, uint32_t *__restrict__ counters,
    LongRow *__restrict__ longs, uint2 *__restrict__ piece_at) {
  constexpr uint32_t kRows = 2, kTerms = 4;
  const uint32_t lane = threadIdx.x & 63u, sub = threadIdx.x / lpr, cl = threadIdx.x % lpr,
                 per = 256 / lpr, in_wave = min(lpr, 64u);
  for (uint64_t first = (uint64_t)blockIdx.x * (per * kRows); first < rows;
       first += (uint64_t)gridDim.x * per * kRows) {
    uint32_t from[kRows], cnt[kRows];
    uint64_t row[kRows];
#pragma unroll
    for (uint32_t k = 0; k < kRows; ++k) {
      row[k] = first + sub * kRows + k;
      from[k] = row[k] < rows ? start[row[k]] : 0u;
      cnt[k] = row[k] < rows ? start[row[k] + 1] : 0u;
    }
    uint32_t most = 0;
#pragma unroll
    for (uint32_t k = 0; k < kRows; ++k) {
      cnt[k] -= from[k];
      if (cnt[k] > kLong) {
        const uint32_t pieces = ceil_div(cnt[k], kPiece);
        uint32_t at = 0;
        if (cl == 0) {
          at = atomicAdd(&counters[1], pieces);
          longs[atomicAdd(&counters[0], 1u)] = LongRow{(uint32_t)row[k], at};
        }
        if (cl < 64) {  // the lanes of the group that share a wave with its first
          at = __shfl(at, lane - cl % in_wave, 64);
          for (uint32_t i = cl; i < pieces; i += in_wave) {
            const uint32_t f = from[k] + i * kPiece;
            piece_at[at + i] = make_uint2(f, f + min(kPiece, from[k] + cnt[k] - f));
          }
        }
        row[k] = rows;  // not here
        cnt[k] = 0;
      }
      most = max(most, cnt[k]);
    }
    for (uint32_t c = cl; c < vecs; c += lpr) {
      const T *const col = dout + (uint64_t)c * V;
      float acc[kRows][V] = {};
      for (uint32_t i = 0; i < most; i += kTerms) {
        uint32_t p[kRows][kTerms];
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k)
#pragma unroll
          for (uint32_t j = 0; j < kTerms; ++j) p[k][j] = i + j < cnt[k] ? pos[from[k] + i + j] : 0u;
        float v[kRows][kTerms][V];
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k)
#pragma unroll
          for (uint32_t j = 0; j < kTerms; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[k][j][e] = 0.f;
            if (i + j < cnt[k]) load_f32<T, V>(col + (uint64_t)p[k][j] * dout_stride, v[k][j]);
          }
#pragma unroll
        for (uint32_t k = 0; k < kRows; ++k)
#pragma unroll
          for (uint32_t j = 0; j < kTerms; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) acc[k][e] += v[k][j][e];
      }
#pragma unroll
      for (uint32_t k = 0; k < kRows; ++k) {
        if (row[k] >= rows) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[k][e] *= scale;
        store_f32<G, V>(dtable + row[k] * table_stride + (uint64_t)c * V, acc[k]);
      }
    }
  }
}

// One wave per piece and 64 column vectors; part: pieces x width, in float64:
// a crowded row may have tens of thousands of terms
template <typename T, int V>
__global__ __launch_bounds__(64) void k_embed_pieces(const T *__restrict__ dout,
                                                     uint64_t dout_stride,
                                                     const uint32_t *__restrict__ pos,
                                                     const uint32_t *__restrict__ counters,
                                                     const uint2 *__restrict__ piece_at,
                                                     double *__restrict__ part, uint32_t vecs,
                                                     uint32_t width) {
  const uint32_t n = counters[1];
  const uint32_t c = blockIdx.y * 64 + threadIdx.x;
  if (c >= vecs) return;
  for (uint32_t k = blockIdx.x; k < n; k += gridDim.x) {
    const uint2 at = piece_at[k];
    double acc[V] = {};
    add_terms<T, V>(dout + (uint64_t)c * V, dout_stride, pos, at.x, at.y, acc);
#pragma unroll
    for (int j = 0; j < V; ++j) part[(uint64_t)k * width + c * V + j] = acc[j];
  }
}

// The crowded rows: 16 waves each add a run of a row's pieces, then the
// runs' sums are added in order.
template <typename G>
__global__ __launch_bounds__(1024) void k_embed_join(const uint32_t *__restrict__ counters,
                                                     const LongRow *__restrict__ longs,
                                                     const uint32_t *__restrict__ start,
                                                     const double *__restrict__ part,
                                                     G *__restrict__ dtable, uint64_t table_stride,
                                                     uint32_t width, float scale) {
  __shared__ double s_sum[16][64];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t n = counters[0];
  const uint32_t c = blockIdx.y * 64 + lane;
  for (uint32_t k = blockIdx.x; k < n; k += gridDim.x) {
    const LongRow lr = longs[k];
    const uint32_t pieces = ceil_div(start[lr.row + 1] - start[lr.row], kPiece);
    const uint32_t run = ceil_div(pieces, 16);
    const uint32_t a = min(wave * run, pieces), b = min(a + run, pieces);
    double acc = 0.0;
    if (c < width)
      for (uint32_t p = a; p < b; ++p) acc += part[(uint64_t)(lr.piece + p) * width + c];
    s_sum[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < width) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < 16; ++w) t += s_sum[w][lane];
      const float o[1] = {(float)(t * scale)};
      store_f32<G, 1>(dtable + (uint64_t)lr.row * table_stride + c, o);
    }
    __syncthreads();
  }
}

// ---- workspace of the gradient

struct GradPlan {
  uint64_t keys, vals, keys2, vals2, hist, totals, start, counters, longs, pieces, part, total;
  uint32_t long_max, piece_max, tiles, digits;
  int passes, bits;  // of a pass
  bool whole;        // one pass, a digit a whole key
};


GradPlan grad_plan(const nsfps_embed_args &a) {
  GradPlan p;
  uint64_t off = 0;
  const auto take = [&](uint64_t bytes) {
    const uint64_t at = off;
    off = (off + bytes + 255) & ~255ull;
    return at;
  };
  int bits = 1;
  while (bits < 32 && (a.rows >> bits)) ++bits;  // keys 0 .. rows
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  // One pass over whole keys where their counts fit LDS and the histograms
  // (one a tile) stay small.  us a gradient of 64 columns, in passes of 10 bits
  // and in one: 1,000 tokens of 8,192 rows 41, 20; 16,384 of 1,000 46, 37;
  // 16,384 of 12,000 48, 33; 262,144 of 12,000 220, 208.
  p.whole = a.rows < kPlaceDigits && a.tokens <= 256 * kPlaceTile;
  p.tiles = (uint32_t)host_ceil_div(a.tokens, p.whole ? kPlaceTile : kTokTile);
  if (p.whole) p.passes = 1, p.bits = bits;
  p.digits = p.whole ? (uint32_t)a.rows + 1 : 1u << p.bits;
  p.long_max = (uint32_t)(a.tokens / (kLong + 1));
  p.piece_max = (uint32_t)(a.tokens / kPiece) + p.long_max;
  p.keys = take(4 * a.tokens);
  p.vals = take(4 * a.tokens);
  p.keys2 = take(4 * a.tokens);
  p.vals2 = take(4 * a.tokens);
  p.hist = take(4ull * p.tiles * p.digits);
  p.totals = take(4ull * p.digits);
  p.start = take(4 * (a.rows + 1));
  p.counters = take(8);
  p.longs = take(sizeof(LongRow) * (uint64_t)p.long_max);
  p.pieces = take(8 * (uint64_t)p.piece_max);
  p.part = take(8ull * p.piece_max * a.width);
  p.total = off;
  return p;
}

template <typename T, typename G, int V>
hipError_t run_grad(const nsfps_embed_args &a, hipStream_t st) {
  const GradPlan p = grad_plan(a);
  char *const w = (char *)a.workspace;
  uint32_t *const counters = (uint32_t *)(w + p.counters), *const start = (uint32_t *)(w + p.start);
  const uint32_t count = (uint32_t)a.tokens, rows = (uint32_t)a.rows;
  uint32_t *keys = nullptr, *pos = nullptr;
  uint32_t *const key_buf[2] = {(uint32_t *)(w + p.keys), (uint32_t *)(w + p.keys2)};
  uint32_t *const pos_buf[2] = {(uint32_t *)(w + p.vals), (uint32_t *)(w + p.vals2)};
  uint32_t *const hist = (uint32_t *)(w + p.hist), *const totals = (uint32_t *)(w + p.totals);
  const bool few = !p.whole && count <= kRankTokens;
  if (few && count) {
    keys = key_buf[0];
    pos = pos_buf[0];
    k_token_rank<<<1, kRankTokens, 0, st>>>(a.d_tokens, keys, pos, count, rows, counters);
  }
  for (int pass = 0; pass < p.passes && count && !few; ++pass) {
    const int shift = pass * p.bits;
    if (p.whole) {
      const hipError_t e = hipFuncSetAttribute(
          (const void *)k_token_place, hipFuncAttributeMaxDynamicSharedMemorySize,
          (int)place_lds(kPlaceDigits));
      if (e != hipSuccess) return e;
      pos = pos_buf[0];
      k_token_hist<kPlaceTile, kPlaceTile><<<p.tiles, kPlaceTile, 4 * p.digits, st>>>(
          a.d_tokens, nullptr, count, rows, 0, p.digits, ~0u, hist, counters);
      k_token_scan<<<(p.digits + 63) / 64, 1024, 0, st>>>(hist, p.tiles, p.digits, totals);
      k_token_place<<<p.tiles, kPlaceThreads, place_lds(p.digits), st>>>(
          a.d_tokens, pos, count, rows, p.bits, hist, totals, start);
      break;
    }
    k_token_hist<256, kTokTile><<<p.tiles, 256, 4 * p.digits, st>>>(
        a.d_tokens, keys, count, rows, shift, p.digits, p.digits - 1, hist, counters);
    k_token_scan<<<(p.digits + 63) / 64, 1024, 0, st>>>(hist, p.tiles, p.digits, totals);
    k_token_scatter<<<p.tiles, 256, 0, st>>>(a.d_tokens, keys, pos, key_buf[pass & 1],
                                             pos_buf[pass & 1], count, rows, shift, p.bits, hist,
                                             totals);
    keys = key_buf[pass & 1];
    pos = pos_buf[pass & 1];
  }
  if (!p.whole || !count)
    k_embed_starts<<<(uint32_t)host_ceil_div((uint64_t)count + 1, 256), 256, 0, st>>>(keys, count,
                                                                                     rows, start);
  const uint32_t vecs = a.width / V;
  const T *dout = (const T *)a.d_out;
  G *dtable = (G *)a.d_table;
  LongRow *const longs = (LongRow *)(w + p.longs);
  uint2 *const pieces = (uint2 *)(w + p.pieces);
  double *const part = (double *)(w + p.part);
  uint32_t lpr = 1;
  while (lpr < 256 && lpr < vecs) lpr *= 2;
  const uint64_t per_group = 2 * (256 / lpr);  // two rows a lane group
  k_embed_rows<T, G, V><<<grid_of(host_ceil_div(rows, per_group)), 256, 0, st>>>(
      dout, a.out_stride, pos, start, dtable, a.table_stride, rows, vecs, lpr, a.scale, counters,
      longs, pieces);
  if (p.long_max) {
    const dim3 gp(std::min(p.piece_max, 4096u), (uint32_t)host_ceil_div(vecs, 64));
    k_embed_pieces<T, V><<<gp, 64, 0, st>>>(dout, a.out_stride, pos, counters, pieces, part, vecs,
                                            a.width);
    const dim3 gj(std::min(p.long_max, 512u), (uint32_t)host_ceil_div(a.width, 64));
    k_embed_join<G><<<gj, 1024, 0, st>>>(counters, longs, start, part, dtable, a.table_stride,
                                         a.width, a.scale);
  }
  return hipGetLastError();
}

bool wide_table(const void *p, uint64_t stride, uint32_t width, uint32_t v, uint32_t size) {
  return (uintptr_t)p % (v * size) == 0 && stride % v == 0 && width % v == 0;
}

}  // namespace

hipError_t launch_embed(const nsfps_embed_args &a, hipStream_t st) {
  const auto go = [&](auto *t, auto v) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int V = decltype(v)::value;
    const uint32_t vecs = a.width / V;
    uint32_t tpr = 1;
    while (tpr < 256 && tpr < vecs) tpr *= 2;
    k_embed<T, V><<<grid_of(host_ceil_div(a.tokens, 256 / tpr)), 256, 0, st>>>(
        (const T *)a.d_table, a.d_tokens, (T *)a.d_out, (uint32_t)a.tokens, (uint32_t)a.rows, vecs,
        a.table_stride, a.out_stride, a.scale, tpr);
    return hipGetLastError();
  };
  const uint32_t size = a.dtype == NSFPS_F32 ? 4 : 2, v = 16 / size;
  const bool wide = wide_table(a.d_table, a.table_stride, a.width, v, size) &&
                    wide_table(a.d_out, a.out_stride, a.width, v, size);
  if (a.dtype == NSFPS_F32)
    return wide ? go((float *)nullptr, std::integral_constant<int, 4>())
                : go((float *)nullptr, std::integral_constant<int, 1>());
  return wide ? go((bf16 *)nullptr, std::integral_constant<int, 8>())
              : go((bf16 *)nullptr, std::integral_constant<int, 1>());
}

uint64_t embed_grad_bytes(const nsfps_embed_args &a) { return grad_plan(a).total; }

hipError_t launch_embed_grad(const nsfps_embed_args &a, hipStream_t st) {
  const bool tf = a.dtype == NSFPS_F32, gf = a.grad_dtype == NSFPS_F32;
  const uint32_t ts = tf ? 4 : 2, gs = gf ? 4 : 2;
  // 16 bytes of the wider type a lane, where both sides' rows allow it
  const auto fits = [&](uint32_t v) {
    return wide_table(a.d_out, a.out_stride, a.width, v, ts) &&
           wide_table(a.d_table, a.table_stride, a.width, v, gs);
  };
  if (tf)
    return gf ? (fits(4) ? run_grad<float, float, 4>(a, st) : run_grad<float, float, 1>(a, st))
              : (fits(4) ? run_grad<float, bf16, 4>(a, st) : run_grad<float, bf16, 1>(a, st));
  if (gf) return fits(4) ? run_grad<bf16, float, 4>(a, st) : run_grad<bf16, float, 1>(a, st);
  return fits(8) ? run_grad<bf16, bf16, 8>(a, st) : run_grad<bf16, bf16, 1>(a, st);
}

hipError_t preload_embed_kernels() {
  return func_attributes(k_embed<bf16, 8>, k_embed<bf16, 1>, k_embed<float, 4>, k_embed<float, 1>,
                         k_token_hist<256, kTokTile>,
                         k_token_hist<kPlaceTile, kPlaceTile>, k_token_scan, k_token_scatter, k_token_place, k_token_rank, k_embed_starts,
                         k_embed_rows<bf16, bf16, 8>,
                         k_embed_rows<float, float, 4>);
}

}  // namespace nsfps
