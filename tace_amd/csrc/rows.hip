// Row operators: table lookup by token with its gradient, rows sorted by
// expert and back.  All of them move rows once and are bound by HBM (a copy of
// 4 GiB reaches 4.8 TB/s here, one of 64 MiB 6.9, a fill 6.9), small ones by
// their launches.
#include "../../include/tace_hip.h"
#include "row_types.h"

#include <algorithm>

namespace {

// ------------------------------------------------------------- embedding ----
constexpr int WG = 256;
constexpr int MAX_ROW = 1 << 15;   // elements: RowDiv's range

// A chunk of a row for each thread, in order.
struct RowChunks {
  int64_t total;      // rows * chunks
  RowDiv chunks;      // chunks a row

  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int64_t q0 = (int64_t)blockIdx.x * WG, r0 = q0 / chunks.d;
    const unsigned rem = (unsigned)(q0 - r0 * chunks.d), q = rem + threadIdx.x;
    if (q0 + threadIdx.x < total) {
      const unsigned r = chunks.div(q);
      f(r0 + r, q - r * chunks.d);
    }
  }
};

// out[i] = scale table[tokens[i]], zeros outside the table.  The table stays in
// L2; bound by the stores, which go past the caches: 1.06 M rows of 64 float32
// (272 MB) 44 us, 6.3 TB/s (57 with four chunks a thread and stores that stay
// in the caches, 47 with two and stores past them).
template <typename T, int V, typename I>
__global__ __launch_bounds__(WG) void k_embed_fwd(const T* __restrict__ table, const I* __restrict__ tokens,
                                                  RowChunks rc, int64_t vocab, row_sum_t<T> scale,
                                                  T* __restrict__ out) {
  typedef row_vec_t<T, V> Vec;
  const Vec* tab = (const Vec*)table;
  Vec* o = (Vec*)out;
  rc.each([&](int64_t r, unsigned c) {
    const I t = tokens[r];
    row_sum_t<T> a[V];
    if (t >= 0 && t < (I)vocab) {
      row_widen<T, V>(tab[(int64_t)t * rc.chunks.d + c], a);
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] *= scale;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = 0;
    }
    __builtin_nontemporal_store(row_round<T, V>(a), &o[r * rc.chunks.d + c]);
  });
}

// The gradient by sorted tokens.  A workgroup takes `per` sorted positions for
// each of its groups of `lanes` threads, which hold a row's sums in registers.
// Sorted, a token's rows are a run; whether a run goes on outside a group's (or
// the workgroup's) positions shows in the neighbouring position's token.  Runs
// inside a group are written at once; the others meet in LDS, in position order,
// a team of groups first.
//
// `Src` says what the sorted positions are:
//   at(p)        the row of sorted position p (any p; the nearest one outside)
//   key(p, row)  its token, -1 behind the last (padding)
//   left(), right()  the tokens before and behind the workgroup's positions, -1: none
//   whole(v, c, sum), open(v, slot, c, sum)  where the sum of a run goes that
//       ends inside the workgroup, and of one that goes on (slot 0: began before it)
// Bound by rows read in no order, past the caches, eight in flight a thread while
// the next eight positions are looked up: 1.06 M rows of 64 float32 of 7,921
// tokens 61 us, 4.5 TB/s (70 through the caches; four or sixteen in flight are
// within 3%).  Joining all groups' runs by one group, not by teams, made 1 M rows
// of 16 float32 47 us instead of 37: 128 sums in sequence.
constexpr int TEAM = 8;   // groups whose open runs one of them joins
template <typename T, int V>
struct RunSums {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  S open[2 * V * WG];   // [slot][element][thread]
  int open_key[2 * WG], team_key[2 * WG / TEAM], outer[2 * WG / TEAM];

  template <typename Src>
  __device__ __forceinline__ void run(const Src& src, const T* __restrict__ g, int cw, int lanes, int p_begin,
                                      int p_end, int per) {
    constexpr int U = 8;
    const int groups = WG / lanes, t = (int)threadIdx.x;
    const int grp = t / lanes, lane = t % lanes, c = lane + (int)blockIdx.y * lanes;
    const int p0 = (int)min(p_begin + (int64_t)grp * per, (int64_t)p_end);
    const int p1 = (int)min((int64_t)p0 + per, (int64_t)p_end);
    if (grp < groups) {
      int next[U];
      auto ahead = [&](int p) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = src.at(p + u);
      };
      ahead(p0);
      const int left = p0 > p_begin ? src.key(p0 - 1, src.at(p0 - 1)) : src.left();
      const int right = p1 < p_end ? src.key(p1, src.at(p1)) : src.right();
      if (lane == 0) {
        const int team = grp / TEAM;
        open_key[2 * grp] = open_key[2 * grp + 1] = -1;
        if (grp % TEAM == 0) outer[2 * team] = left, team_key[2 * team] = team_key[2 * team + 1] = -1;
        if (grp % TEAM == TEAM - 1 || grp == groups - 1) outer[2 * team + 1] = right;
      }
      S sum[V];
      int cur = -1;
      bool head = true;   // the run at p0
      auto flush = [&]() {
        if (cur < 0 || c >= cw) return;
        if (cur != left && cur != right) {
          src.whole(cur, c, sum);
        } else {
          const int slot = head ? 0 : 1;
#pragma unroll
          for (int i = 0; i < V; ++i) open[(slot * V + i) * WG + t] = sum[i];
          if (lane == 0) open_key[2 * grp + slot] = cur;
        }
      };
      const Vec* rows = (const Vec*)g + min(c, cw - 1);
      for (int p = p0; p < p1; p += U) {
        int at[U];
        Vec v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          at[u] = next[u];
          v[u] = __builtin_nontemporal_load(rows + (int64_t)at[u] * cw);   // (read once)
        }
        int key[U];
#pragma unroll
        for (int u = 0; u < U; ++u) key[u] = src.key(p + u, at[u]);
        ahead(p + U);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int k = p + u < p1 ? key[u] : cur;
          S a[V];
          row_widen<T, V>(v[u], a);
          if (k != cur) {
            flush();
            head = head && cur < 0;
            cur = k;
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = a[i];
          } else if (p + u < p1) {
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += a[i];
          }
        }
      }
      flush();
    }
    __syncthreads();
    // the open runs of `count` groups, `step` apart, from g0 on
    auto merge = [&](int g0, int count, int step, const int* keys, int left, int right, auto&& leave) {
      S sum[V];
      int cur = -1;
      auto flush = [&]() {
        if (cur != left && cur != right) src.whole(cur, c, sum);
        else leave(cur == left ? 0 : 1, cur, sum);
      };
      for (int q = 0; q < 2 * count; ++q) {
        const int key = keys[q];
        if (key < 0) continue;
        const S* o = open + (q & 1) * V * WG + (g0 + (q >> 1) * step) * lanes + lane;
        if (key != cur) {
          if (cur >= 0) flush();
          cur = key;
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] = o[i * WG];
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) sum[i] += o[i * WG];
        }
      }
      if (cur >= 0) flush();
    };
    const int teams = (groups + TEAM - 1) / TEAM;
    auto leave_open = [&](int slot, int v, const S* sum) { src.open(v, slot, c, sum); };
    if (teams == 1) {
      if (grp == 0 && c < cw) merge(0, groups, 1, open_key, outer[0], outer[1], leave_open);
      return;
    }
    // (a thread reads and writes its own sums here, and those of its column in its team)
    if (grp < groups && grp % TEAM == 0 && c < cw) {
      const int team = grp / TEAM;
      merge(grp, min(TEAM, groups - grp), 1, open_key + 2 * grp, outer[2 * team], outer[2 * team + 1],
            [&](int slot, int key, const S* sum) {
#pragma unroll
              for (int i = 0; i < V; ++i) open[(slot * V + i) * WG + t] = sum[i];
              if (lane == 0) team_key[2 * team + slot] = key;
            });
    }
    __syncthreads();
    if (grp == 0 && c < cw) merge(0, teams, TEAM, team_key, outer[0], outer[2 * teams - 1], leave_open);
  }
};

// Positions sorted ahead (order): a run that goes on beyond the workgroup is
// left in part [workgroup][slot][channels], for k_embed_grad_join.
template <typename T, int V, typename I>
struct SortedRows {
  const I* tokens;
  const int* order;
  int n, vocab, channels, p_begin, p_end;
  row_sum_t<T> scale;
  T* grad;
  row_sum_t<T>* part;

  // (positions of another grouping than these tokens' stay inside the rows)
  __device__ __forceinline__ int at(int p) const {
    return (int)min((unsigned)order[min(max(p, 0), n - 1)], (unsigned)n - 1);
  }
  __device__ __forceinline__ int key(int, int row) const {
    const I v = tokens[row];
    return v >= 0 && v < (I)vocab ? (int)v : -1;
  }
  __device__ __forceinline__ int left() const { return p_begin > 0 ? key(0, at(p_begin - 1)) : -1; }
  __device__ __forceinline__ int right() const { return p_end < n ? key(0, at(p_end)) : -1; }
  __device__ __forceinline__ void whole(int v, int c, const row_sum_t<T>* sum) const {
    row_sum_t<T> a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) a[i] = sum[i] * scale;
    ((row_vec_t<T, V>*)grad)[(int64_t)v * (channels / V) + c] = row_round<T, V>(a);
  }
  __device__ __forceinline__ void open(int, int slot, int c, const row_sum_t<T>* sum) const {
    row_sum_t<T>* o = part + ((int64_t)blockIdx.x * 2 + slot) * channels + (int64_t)c * V;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = sum[i];
  }
};

template <typename T, int V, typename I>
__global__ __launch_bounds__(WG) void k_embed_grad_part(const T* __restrict__ g, const I* __restrict__ tokens,
                                                        const int* __restrict__ order, int n, int vocab, int channels,
                                                        int per, int lanes, row_sum_t<T> scale, T* __restrict__ grad,
                                                        row_sum_t<T>* __restrict__ part) {
  __shared__ RunSums<T, V> sums;
  const int64_t span = (int64_t)per * (WG / lanes), w0 = blockIdx.x * span;
  const int p0 = (int)min(w0, (int64_t)n), p1 = (int)min(w0 + span, (int64_t)n);
  const SortedRows<T, V, I> src{tokens, order, n, vocab, channels, p0, p1, scale, grad, part};
  sums.run(src, g, channels / V, lanes, p0, p1, per);
}

// Few tokens (at most 128): a workgroup sorts its own `rows` rows' tokens in
// LDS, so no grouping of all of them is needed; each token's sum goes to part
// [workgroup][token][channels] and its presence to seen [workgroup][token], for
// k_embed_grad_total.  Two launches instead of four; bound by the chain of loads
// of a workgroup: 101,306 rows of 128 bfloat16 of two tokens 13.9 us and 3.9 for
// the total.
//
// More tokens in buckets of 128: the rows are grouped by bucket first (order,
// bptr [buckets + 1]; few keys, two launches) and a workgroup has rows of one
// bucket.  first [buckets + 1]: each bucket's first workgroup.  1.06 M rows of 64
// float32 of 7,921 tokens: 19 us to group them, 71 here, 11 for the total.
constexpr int FEW_TOKENS = 128, BUCKET_BITS = 7, LOCAL_STEPS = 10, LOCAL_ROWS = WG * LOCAL_STEPS, MAX_BUCKETS = 255;
template <typename T, int V, bool BUCKETS>
struct LocalRows {
  const int* list;    // token << 16 | row in the workgroup, sorted
  const int* rowid;   // BUCKETS: the rows
  int64_t row0;
  int count, width, channels;
  row_sum_t<T>* part;

  __device__ __forceinline__ int packed(int p) const { return list[min(max(p, 0), count - 1)]; }
  __device__ __forceinline__ int at(int p) const {
    const int i = packed(p) & 0xffff;
    return BUCKETS ? rowid[i] : (int)(row0 + i);
  }
  __device__ __forceinline__ int key(int p, int) const { return p < count ? packed(p) >> 16 : -1; }
  __device__ __forceinline__ int left() const { return -1; }
  __device__ __forceinline__ int right() const { return -1; }
  __device__ __forceinline__ void whole(int v, int c, const row_sum_t<T>* sum) const {
    row_sum_t<T>* o = part + ((int64_t)blockIdx.x * width + v) * channels + (int64_t)c * V;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = sum[i];
  }
  __device__ __forceinline__ void open(int, int, int, const row_sum_t<T>*) const {}   // (no run goes on)
};

// Bucket of this workgroup and its first and last position: the buckets' counts
// of workgroups are summed by every workgroup (at most 255 of them).  False for
// a workgroup too many.
__device__ __forceinline__ bool bucket_of(const int* __restrict__ bptr, int buckets, int rows, int* __restrict__ first,
                                          int* found, int* wsum, int* bucket, int* begin, int* end) {
  const int t = (int)threadIdx.x, lane = t & 63, w = t >> 6;
  const int a = t < buckets ? bptr[t] : 0, z = t < buckets ? bptr[t + 1] : 0;
  const int wgs = (z - a + rows - 1) / rows;
  int inc = wgs;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (lane == 63) wsum[w] = inc;
  if (t == 0) found[0] = -1;
  __syncthreads();
  for (int k = 0; k < w; ++k) inc += wsum[k];
  const int at = inc - wgs;   // this bucket's first workgroup
  if (blockIdx.x == 0 && blockIdx.y == 0 && t <= buckets) first[t] = at;   // (t = buckets: all of them)
  if ((int)blockIdx.x >= at && (int)blockIdx.x < inc) {
    found[0] = t;
    found[1] = a + ((int)blockIdx.x - at) * rows;
    found[2] = min(found[1] + rows, z);
  }
  __syncthreads();
  *bucket = found[0];
  *begin = found[1];
  *end = found[2];
  return *bucket >= 0;
}

template <typename T, int V, typename I, bool BUCKETS>
__global__ __launch_bounds__(WG) void k_embed_grad_local(const T* __restrict__ g, const I* __restrict__ tokens,
                                                         const int* __restrict__ order, const int* __restrict__ bptr,
                                                         int buckets, int n, int vocab, int channels, int rows,
                                                         int lanes, int* __restrict__ first, int* __restrict__ seen,
                                                         row_sum_t<T>* __restrict__ part) {
  constexpr int WAVES = WG / 64;
  __shared__ RunSums<T, V> sums;
  __shared__ int list[LOCAL_ROWS], rowid[BUCKETS ? LOCAL_ROWS : 1], cnt[WAVES][FEW_TOKENS], wsum[WAVES], found[3], kept;
  const int t = (int)threadIdx.x, lane = t & 63, w = t >> 6, steps = rows / WG;
  int bucket = 0, begin = 0, end = 0;
  if constexpr (BUCKETS) {
    if (!bucket_of(bptr, buckets, rows, first, found, wsum, &bucket, &begin, &end)) return;
  }
  const int64_t row0 = BUCKETS ? begin : (int64_t)blockIdx.x * rows, stop = BUCKETS ? end : n;
  const int width = BUCKETS ? FEW_TOKENS : vocab, base = bucket << BUCKET_BITS;
  for (int q = t; q < WAVES * FEW_TOKENS; q += WG) cnt[q / FEW_TOKENS][q % FEW_TOKENS] = 0;
  const int i0 = 64 * steps * w + lane;   // (of the workgroup's rows; a run of 64 `steps` a wavefront)
  I tok[LOCAL_STEPS];
  int row[LOCAL_STEPS];
#pragma unroll
  for (int u = 0; u < LOCAL_STEPS; ++u)
    if (u < steps) {
      const int p = (int)min(row0 + i0 + 64 * u, stop - 1);
      row[u] = BUCKETS ? order[p] : p;
    }
#pragma unroll
  for (int u = 0; u < LOCAL_STEPS; ++u)
    if (u < steps) {
      tok[u] = tokens[row[u]];
      if (BUCKETS) rowid[i0 + 64 * u] = row[u];
    }
  __syncthreads();
  int key[LOCAL_STEPS], rank[LOCAL_STEPS];
#pragma unroll
  for (int u = 0; u < LOCAL_STEPS; ++u) {
    const bool in = u < steps && row0 + i0 + 64 * u < stop && tok[u] >= 0 && tok[u] < (I)vocab;
    key[u] = in ? (int)tok[u] - base : -1;   // (0 .. 127)
    if (u >= steps) continue;   // (all lanes alike)
    unsigned long long m = __ballot(in);
#pragma unroll
    for (int b = 0; b < BUCKET_BITS; ++b) {
      const bool one = (key[u] >> b) & 1;
      const unsigned long long v = __ballot(one);
      m &= one ? v : ~v;
    }
    const int r = __popcll(m & ((1ull << lane) - 1));
    int had = 0;
    if (in && r == 0) had = atomicAdd(&cnt[w][key[u]], __popcll(m));
    rank[u] = r + __shfl(had, in ? __ffsll((long long)m) - 1 : lane, 64);
  }
  __syncthreads();
  int sum = 0;
  if (t < FEW_TOKENS)
    for (int k = 0; k < WAVES; ++k) sum += cnt[k][t];
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (w < 2 && lane == 63) wsum[w] = inc;
  __syncthreads();
  if (t < FEW_TOKENS) {
    int at = inc - sum + (w == 1 ? wsum[0] : 0);
    if (t == FEW_TOKENS - 1) kept = at + sum;
    if (t < width && blockIdx.y == 0) seen[(int64_t)blockIdx.x * width + t] = sum;
    for (int k = 0; k < WAVES; ++k) {
      const int c = cnt[k][t];
      cnt[k][t] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < LOCAL_STEPS; ++u)
    if (key[u] >= 0) list[cnt[w][key[u]] + rank[u]] = key[u] << 16 | (i0 + 64 * u);
  __syncthreads();
  const int count = kept;
  if (count == 0) return;
  const LocalRows<T, V, BUCKETS> src{list, rowid, row0, count, width, channels, part};
  const int groups = WG / lanes;
  sums.run(src, g, channels / V, lanes, 0, count, (count + groups - 1) / groups);
}

// What is left: workgroup w < workgroups - 1 joins the run that begins in the
// w-th workgroup above and goes on in the next (if there is one); the others
// write the zeros of tokens without rows, one per wavefront and step.
constexpr int JOIN_COLS = 16, JOIN_ROWS = WG / JOIN_COLS;
template <typename T, typename I>
__global__ __launch_bounds__(WG) void k_embed_grad_join(const I* __restrict__ tokens, const int* __restrict__ order,
                                                        const int* __restrict__ rowptr, int n, int vocab,
                                                        int channels, int64_t span, int seams, row_sum_t<T> scale,
                                                        const row_sum_t<T>* __restrict__ part, T* __restrict__ grad) {
  typedef row_sum_t<T> S;
  const int t = (int)threadIdx.x;
  if ((int)blockIdx.x >= seams) {
    const int step = ((int)gridDim.x - seams) * (WG / 64) * (int)gridDim.y;
    const int first = (((int)blockIdx.x - seams) * (int)gridDim.y + (int)blockIdx.y) * (WG / 64) + t / 64;
    for (int64_t v = first; v < vocab; v += step)
      if (rowptr[v] == rowptr[v + 1])
        for (int c = t % 64; c < channels; c += 64) grad[v * channels + c] = (T)0;
    return;
  }
  const int64_t w0 = blockIdx.x * span, w1 = w0 + span;   // (w1 < n)
  const I tok = tokens[min((unsigned)order[w1], (unsigned)n - 1)];
  if (tok < 0 || tok >= (I)vocab) return;   // padding
  const int v = (int)tok, b = rowptr[v], e = min(rowptr[v + 1], n);
  if (b >= w1 || b < w0) return;   // begins at the seam, or joined at an earlier one
  __shared__ S red[JOIN_ROWS][JOIN_COLS];
  const int x = t % JOIN_COLS, y = t / JOIN_COLS, c = (int)blockIdx.y * JOIN_COLS + x;
  const int last = (int)((e - 1) / span);
  S sum = 0;
  if (c < channels) {
#pragma unroll 8
    for (int q = (int)blockIdx.x + y; q <= last; q += JOIN_ROWS)
      sum += part[((int64_t)q * 2 + (q == (int)blockIdx.x ? 1 : 0)) * channels + c];
  }
  red[y][x] = sum;
  __syncthreads();
  if (y == 0 && c < channels) {
#pragma unroll
    for (int k = 1; k < JOIN_ROWS; ++k) sum += red[k][x];
    grad[(int64_t)v * channels + c] = (T)(sum * scale);
  }
}

// grad of k_embed_grad_local's sums: COLS columns of a token for each WG / TOKENS
// threads.  Without buckets there are few tokens and many sums of each; with
// them (first) many tokens, most of few sums.
template <typename T, int COLS, int TOKENS>
__global__ __launch_bounds__(WG) void k_embed_grad_total(const int* __restrict__ seen, const int* __restrict__ first,
                                                         int workgroups, int vocab, int channels, row_sum_t<T> scale,
                                                         const row_sum_t<T>* __restrict__ part, T* __restrict__ grad) {
  typedef row_sum_t<T> S;
  constexpr int ROWS = WG / COLS / TOKENS;
  __shared__ S red[TOKENS * ROWS][COLS];
  const int t = (int)threadIdx.x, x = t % COLS, yy = t / COLS, y = yy % ROWS;
  const int v = (int)blockIdx.x * TOKENS + yy / ROWS, c = (int)blockIdx.y * COLS + x;
  const int bucket = v >> BUCKET_BITS, width = first ? FEW_TOKENS : vocab, at = first ? v % FEW_TOKENS : v;
  S sum = 0;
  if (c < channels && v < vocab) {
    const int q0 = first ? first[bucket] : 0, q1 = first ? first[bucket + 1] : workgroups;
#pragma unroll 8
    for (int q = q0 + y; q < q1; q += ROWS) {
      const int64_t i = (int64_t)q * width + at;
      const S p = part[i * channels + c];   // (holds nothing where the token was not seen)
      sum += seen[i] ? p : (S)0;
    }
  }
  red[yy][x] = sum;
  __syncthreads();
  if (y == 0 && c < channels && v < vocab) {
#pragma unroll
    for (int k = 1; k < ROWS; ++k) sum += red[yy + k][x];
    grad[(int64_t)v * channels + c] = (T)(sum * scale);
  }
}

// Few rows: a workgroup per token (and tile of columns) lists the token's rows
// in LDS and sums them; no grouping, one launch.  Bound by latency: 1,024 rows of
// 128 float32 of 4 tokens 5.5 us.
constexpr int SCAN_N = 4096;
template <typename T, int V, typename I>
__global__ __launch_bounds__(WG) void k_embed_grad_scan(const T* __restrict__ g, const I* __restrict__ tokens, int n,
                                                        int channels, int lanes, row_sum_t<T> scale,
                                                        T* __restrict__ grad) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  __shared__ int list[SCAN_N], found[WG / 64];
  __shared__ S red[WG * V];
  const int t = (int)threadIdx.x, lane = t & 63, w = t >> 6;
  const I v = (I)blockIdx.x;
  int count = 0;
  for (int base = 0; base < n; base += WG) {
    const int i = base + t;
    const bool hit = i < n && tokens[i] == v;
    const unsigned long long m = __ballot(hit);
    if (lane == 0) found[w] = __popcll(m);
    __syncthreads();
    int at = count;
#pragma unroll
    for (int k = 0; k < WG / 64; ++k) {
      if (k < w) at += found[k];
      count += found[k];
    }
    if (hit) list[at + __popcll(m & ((1ull << lane) - 1))] = i;
    __syncthreads();
  }
  const int cw = channels / V, groups = WG / lanes, grp = t / lanes, c = t % lanes + (int)blockIdx.y * lanes;
  S sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0;
  if (grp < groups && c < cw) {
    const Vec* rows = (const Vec*)g;
#pragma unroll 4
    for (int k = grp; k < count; k += groups) {
      S a[V];
      row_widen<T, V>(rows[(int64_t)list[k] * cw + c], a);
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += a[i];
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) red[i * WG + t] = sum[i];
  __syncthreads();
  if (grp == 0 && c < cw) {
    for (int k = 1; k < groups; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += red[i * WG + t + k * lanes];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] *= scale;
    ((Vec*)grad)[(int64_t)v * cw + c] = row_round<T, V>(sum);
  }
}

// no rows
template <typename T>
__global__ __launch_bounds__(WG) void k_embed_grad_none(int64_t total, T* __restrict__ grad) {
  for (int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x; i < total; i += (int64_t)gridDim.x * WG) grad[i] = (T)0;
}

int embed_lanes(int cw) { return cw < WG ? cw : WG; }

// Positions a group: 512 workgroups, at least 8.  (us of 256, 512, 1,024
// workgroups: 1.06 M rows of 64 float32 73, 63, 69; 200,000 of 256 49, 43, 48;
// 60,000 of 1,000 float16 47, 48, 62: fewer leave CUs idle, more spend their time
// on their first loads and their seams.)
int embed_per(int64_t n, int lanes) {
  const int64_t groups = WG / lanes, per = (n + 512 * groups - 1) / (512 * groups);
  return (int)(per < 8 ? 8 : per);
}
// workgroups for rows of cw chunks, whatever their type
int64_t embed_wgs(int64_t n, int lanes) {
  const int64_t span = (int64_t)embed_per(n, lanes) * (WG / lanes);
  return (n + span - 1) / span;
}

// --------------------------------------------------------------- routing ----
// A row's chunks in blocks that lie apart: block b of R rows starts at R *
// start[b] chunks and holds start[b + 1] - start[b] of each row.
struct Blocks {
  int count;
  unsigned start[TACE_ROW_MAX_BLOCKS + 1];

  __device__ __forceinline__ int64_t at(int64_t rows, int64_t row, unsigned c) const {
    unsigned lo = 0, hi = start[1];
#pragma unroll
    for (int b = 1; b < TACE_ROW_MAX_BLOCKS; ++b)
      if (b < count && c >= start[b]) {
        lo = start[b];
        hi = start[b + 1];
      }
    return rows * lo + row * (hi - lo) + (c - lo);
  }
};

__global__ __launch_bounds__(WG) void k_route_place(const int* __restrict__ order, int n, int* __restrict__ place) {
  const int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x;
  if (i < n) place[order[i]] = (int)i;
}

// Stable grouping by few keys (at most 255, and one for keys outside them): a
// workgroup of 16 wavefronts has 1,024 `steps` positions in runs of 64 `steps`
// a wavefront.  k_few_count leaves its counts of every key; k_few_place adds up
// those of the workgroups before it and of all, ranks its own positions by
// ballots and writes their places.  One workgroup (n <= 8,192) counts for
// itself.  Bound by latency; us, with places | general grouping (tace_group_keys:
// any keys, four launches or more), without: 8,192 slots of 8 experts 9 | 11,
// 24,576 of 8 8 | 17, 200,000 of 255 15 | 24, 1 M of 89 22 | 30.  (256 and more, by
// the general grouping and a launch for the places: 8,192 of 256 19, 200,000 of
// 1,000 37, 1 M of 1,000 57.)
constexpr int FEW_WG = 1024, FEW_STEPS = 8, FEW_KEYS = 256, FEW_WGS = 128;

// keys are the values below `limit`, shifted
struct FewKeys {
  int limit, shift, count;
  template <typename I>
  __device__ __forceinline__ int of(I e) const { return e >= 0 && e < (I)limit ? (int)e >> shift : count; }
};

template <typename I>
__global__ __launch_bounds__(FEW_WG) void k_few_count(const I* __restrict__ keys, int64_t stride, int n, FewKeys fk,
                                                      int steps, int* __restrict__ hist) {
  __shared__ int cnt[FEW_KEYS];
  const int t = (int)threadIdx.x;
  if (t < FEW_KEYS) cnt[t] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * FEW_WG * steps + t;
  I e[FEW_STEPS];
#pragma unroll
  for (int u = 0; u < FEW_STEPS; ++u)
    if (u < steps) e[u] = keys[min(i0 + FEW_WG * u, (int64_t)n - 1) * stride];
#pragma unroll
  for (int u = 0; u < FEW_STEPS; ++u)
    if (u < steps && i0 + FEW_WG * u < n) atomicAdd(cnt + fk.of(e[u]), 1);
  __syncthreads();
  if (t <= fk.count) hist[(int64_t)blockIdx.x * (fk.count + 1) + t] = cnt[t];
}

template <typename I>
__global__ __launch_bounds__(FEW_WG) void k_few_place(const I* __restrict__ keys, int64_t stride, int n, FewKeys fk,
                                                      int steps, int bits, const int* __restrict__ hist,
                                                      int* __restrict__ rowptr, int* __restrict__ order,
                                                      int* __restrict__ place) {
  constexpr int WAVES = FEW_WG / 64;
  __shared__ int cnt[WAVES][FEW_KEYS], red[FEW_WG], before[FEW_KEYS], total[FEW_KEYS], wsum[4];
  const int t = (int)threadIdx.x, lane = t & 63, w = t >> 6, nwg = (int)gridDim.x, K = fk.count + 1;
  for (int q = t; q < WAVES * FEW_KEYS; q += FEW_WG) cnt[q / FEW_KEYS][q % FEW_KEYS] = 0;
  const int64_t i0 = ((int64_t)blockIdx.x * WAVES + w) * 64 * steps + lane;
  I e[FEW_STEPS];
#pragma unroll
  for (int u = 0; u < FEW_STEPS; ++u)
    if (u < steps) e[u] = keys[min(i0 + 64 * u, (int64_t)n - 1) * stride];
  // counts of the workgroups before this one, and of all: 2^bits keys side by
  // side, the workgroups dealt to the threads of a key
  int bef = 0, all = 0;
  if (nwg > 1) {
    const int wide = 1 << bits, key = t & (wide - 1);
    if (key < K)
      for (int g = t >> bits; g < nwg; g += FEW_WG >> bits) {
        const int c = hist[(int64_t)g * K + key];
        all += c;
        bef += g < (int)blockIdx.x ? c : 0;
      }
    for (int o = FEW_WG / 2; o >= wide; o >>= 1) {   // (two sums, one after the other)
      red[t] = bef;
      __syncthreads();
      if (t < o) bef += red[t + o];
      __syncthreads();
      red[t] = all;
      __syncthreads();
      if (t < o) all += red[t + o];
      __syncthreads();
    }
    if (t < K) {
      before[t] = bef;
      total[t] = all;
    }
  }
  __syncthreads();
  int key[FEW_STEPS], rank[FEW_STEPS];
#pragma unroll
  for (int u = 0; u < FEW_STEPS; ++u) {
    const bool in = u < steps && i0 + 64 * u < n;
    key[u] = in ? fk.of(e[u]) : -1;
    if (u >= steps) continue;   // (all lanes alike)
    const int k = key[u];
    // this lane's place among its wavefront's equal keys so far
    unsigned long long m = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const bool one = (k >> b) & 1;
      const unsigned long long v = __ballot(one);
      m &= one ? v : ~v;
    }
    const int r = __popcll(m & ((1ull << lane) - 1));
    int had = 0;
    if (in && r == 0) had = atomicAdd(&cnt[w][k], __popcll(m));
    rank[u] = r + __shfl(had, in ? __ffsll((long long)m) - 1 : lane, 64);
  }
  __syncthreads();
  // a key's first place: all smaller keys, its own in the workgroups and in the
  // wavefronts before
  int own = 0;
  if (t < FEW_KEYS)
    for (int k = 0; k < WAVES; ++k) own += cnt[k][t];
  const int sum = t < K ? (nwg > 1 ? total[t] : own) : 0;
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(inc, o, 64);
    if (lane >= o) inc += v;
  }
  if (w < 4 && lane == 63) wsum[w] = inc;
  __syncthreads();
  if (t < FEW_KEYS) {
    int at = inc - sum;
    for (int k = 0; k < w; ++k) at += wsum[k];
    if (t < K && blockIdx.x == 0) rowptr[t] = at;   // (the last: the end of the others)
    if (nwg > 1 && t < K) at += before[t];
    for (int k = 0; k < WAVES; ++k) {
      const int c = cnt[k][t];
      cnt[k][t] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < FEW_STEPS; ++u) {
    if (key[u] < 0) continue;
    const int i = (int)(i0 + 64 * u), at = cnt[w][key[u]] + rank[u];
    order[at] = i;
    if (place) place[i] = at;
  }
}

// whether few_group takes it, and its workgroups and steps
bool few_fits(int64_t n, int64_t n_keys, int* wgs, int* steps) {
  const int64_t most = n <= FEW_WG * FEW_STEPS ? 1 : FEW_WGS;
  *steps = (int)std::min<int64_t>((n + FEW_WG * most - 1) / (FEW_WG * most), FEW_STEPS);
  const int64_t count = n < 1 ? 0 : (n + FEW_WG * *steps - 1) / (FEW_WG * *steps);
  *wgs = (int)std::min<int64_t>(count, 1 << 20);
  return n >= 1 && n_keys < FEW_KEYS && count <= 4 * FEW_WGS;
}

template <typename I>
void few_group(const I* keys, int64_t stride, int n, const FewKeys& fk, int wgs, int steps, int32_t* rowptr,
               int32_t* order, int32_t* place, int32_t* work, hipStream_t s) {
  int bits = 1;
  while ((1 << bits) < fk.count + 1) ++bits;
  if (wgs > 1)
    hipLaunchKernelGGL((k_few_count<I>), dim3((unsigned)wgs), dim3(FEW_WG), 0, s, keys, stride, n, fk, steps, work);
  hipLaunchKernelGGL((k_few_place<I>), dim3((unsigned)wgs), dim3(FEW_WG), 0, s, keys, stride, n, fk, steps, bits, work,
                     rowptr, order, place);
}

// ------------------------------------------- the embedding gradient's form ----
// Which form it takes without a grouping of the tokens: looking through all of
// them, sorting them workgroup by workgroup, that in buckets of 128 tokens, or
// none (it needs a grouping).  us, this form | grouping and sums, float32: SCANS
// 1,024 rows of 128 of 4 tokens 4.7 | 12, 4,096 of 128 of 1,000 tokens 7.5 | 22;
// SORTS 5,000 of 128 of 89 14 | 17, 12,801 of 256 of 89 19 | 20, 101,306 of 128 of 2
// 19 | 30, 1 M of 64 of 89 62 | 77; BUCKETS 9,000 of 64 of 1,000 tokens 23 | 41,
// 50,000 of 64 of 8,000 30 | 47, 1.06 M of 64 of 7,921 95 | 119.  The rule knows
// neither channels nor how full the buckets are, and loses where rows are many
// and wide or buckets few: 1 M of 128 of 128 tokens 124 | 116, 300,000 of 256 of
// 3,000 99 | 98, 1 M of 64 of 300 98 | 98, 300,000 of 64 of 300 55 | 51, 1 M of 128
// of 300 155 | 133.
enum { SCANS = 1, SORTS = 2, BUCKETS = 3, GROUPED = 0 };

// Rows a workgroup (256 .. 2,560) and workgroups, one more a bucket where they
// are not full: about 256 of them, fewer of wide rows, whose columns are dealt to
// several (us of 256, 128, 64: 100,000 rows of 1,000 float32 of 89 tokens 153, 138,
// 116; 300,000 of 256 of 3,000 tokens 104, 109, 109; 101,306 of 128 28, 30, 37).
int local_rows(int64_t n, int32_t channels) {
  const int64_t target = std::min(std::max(65536 / channels, 64), 256);
  const int64_t steps = (n + target * WG - 1) / (target * WG);
  return WG * (int)std::min<int64_t>(std::max<int64_t>(steps, 1), LOCAL_STEPS);
}
int64_t buckets_of(int64_t vocab) { return (vocab + FEW_TOKENS - 1) / FEW_TOKENS; }

int embed_form(int64_t n, int64_t vocab) {
  if (n < 1 || (n <= SCAN_N && vocab <= 1024)) return SCANS;   // (no rows: zeros)
  if (vocab <= FEW_TOKENS) return SORTS;
  int wgs, steps;
  const int64_t buckets = buckets_of(vocab);
  // (its sums are at most about as many as the rows)
  return n > SCAN_N && buckets <= MAX_BUCKETS && buckets * FEW_TOKENS <= n && few_fits(n, buckets, &wgs, &steps)
             ? BUCKETS : GROUPED;
}

// parts of the workspace of SORTS and BUCKETS, in bytes
struct LocalWork {
  int64_t wgs, hist, bptr, order, first, seen, part, bytes;
  LocalWork(int64_t n, int64_t vocab, int32_t channels, int64_t row_bytes) {
    const bool many = vocab > FEW_TOKENS;
    const int64_t buckets = many ? buckets_of(vocab) : 0, width = many ? FEW_TOKENS : vocab;
    const int64_t rows = local_rows(n, channels);
    wgs = (n + rows - 1) / rows + buckets;
    int few = 0, steps = 0;
    if (many) few_fits(n, buckets, &few, &steps);
    bytes = 0;
    auto take = [&](int64_t b) {
      const int64_t at = bytes;
      bytes += (b + 15) / 16 * 16;
      return at;
    };
    hist = take(4 * few * (buckets + 1));
    bptr = take(many ? 4 * (buckets + 1) : 0);
    order = take(many ? 4 * n : 0);
    first = take(many ? 4 * (buckets + 1) : 0);
    seen = take(4 * wgs * width);
    part = take(wgs * width * row_bytes);
  }
};

// STREAM: stores that do not stay in the caches
template <bool STREAM, typename Vec>
__device__ __forceinline__ void put(Vec* p, const Vec& v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// The sorted row of slot s of n: places that are none (of a plan not made by
// tace_route_group) stay inside the rows.  (101,306 x 2 rows of 1,152 bfloat16, both
// directions with gradients, 568 us without and 578 with the bound; 12,288 x 2 of
// 2,048 float32 249 either way.)
__device__ __forceinline__ int place_of(const int* __restrict__ place, int64_t s, int64_t n) {
  return (int)min((unsigned)place[s], (unsigned)n - 1u);
}

// A row is read once and stored k times: 12,288 x 2 rows of 2,048 float32 56 us
// (5.4 TB/s), 101,306 x 2 of 1,152 bfloat16 120 (5.9).
template <typename T, int V, bool STREAM>
__global__ __launch_bounds__(WG) void k_route_dispatch(const T* __restrict__ x, const row_sum_t<T>* __restrict__ w,
                                                       const int* __restrict__ place, const int* __restrict__ rows_end,
                                                       RowChunks rc, int64_t tokens, int k, Blocks bl,
                                                       T* __restrict__ out) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  const int end = *rows_end;
  const int64_t n = tokens * k;
  rc.each([&](int64_t t, unsigned c) {
    const Vec v = ((const Vec*)x)[bl.at(tokens, t, c)];
#pragma unroll 2
    for (int j = 0; j < k; ++j) {
      const int64_t s = t * k + j;
      const int p = place_of(place, s, n);
      Vec o = v;
      if (p >= end || w) {
        S a[V];
        row_widen<T, V>(v, a);
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = p >= end ? (S)0 : a[i] * w[s];
        o = row_round<T, V>(a);
      }
      put<STREAM>((Vec*)out + bl.at(n, p, c), o);
    }
  });
}

// K slots' rows are loaded before the first is added (the dropped ones too:
// they have a row, which is not added): 12,288 x 2 rows of 2,048 float32 53 us (5.7
// TB/s; 60 one after the other), 101,306 x 2 of 1,152 bfloat16 112 (6.1; 131).
template <typename T, int V, int K>
__global__ __launch_bounds__(WG) void k_route_combine(const T* __restrict__ y, const row_sum_t<T>* __restrict__ w,
                                                      const int* __restrict__ place, const int* __restrict__ rows_end,
                                                      RowChunks rc, int64_t tokens, int k, Blocks bl,
                                                      T* __restrict__ out) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  const int end = *rows_end;
  const int64_t n = tokens * k;
  rc.each([&](int64_t t, unsigned c) {
    S sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0;
    for (int j = 0; j < k; j += K) {
      int p[K];
      S f[K];
      Vec v[K];
#pragma unroll
      for (int q = 0; q < K; ++q) {
        const int64_t s = t * k + min(j + q, k - 1);
        p[q] = place_of(place, s, n);
        f[q] = w ? w[s] : (S)1;
      }
#pragma unroll
      for (int q = 0; q < K; ++q) v[q] = ((const Vec*)y)[bl.at(n, p[q], c)];
#pragma unroll
      for (int q = 0; q < K; ++q) {
        if (p[q] >= end || j + q >= k) continue;
        S a[V];
        row_widen<T, V>(v[q], a);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] += f[q] * a[i];
      }
    }
    put<true>((Vec*)out + bl.at(tokens, t, c), row_round<T, V>(sum));
  });
}

// `lanes` (a power of two, at most 64) lanes a slot, the slots of a token side
// by side: its row of x comes from memory once.  U chunks of both rows are
// loaded before the first is multiplied.  12,288 x 2 rows of 2,048 float32 79 us
// (6.4 TB/s; 103 with lanes that take a token's slots one after the other), 1,024
// x 2 of them 10.5 (15), 101,306 x 2 of 1,152 bfloat16 227 (5.2).
template <typename T, int V, int U>
__global__ __launch_bounds__(WG) void k_route_dots(const T* __restrict__ x, const T* __restrict__ y,
                                                   const row_sum_t<T>* __restrict__ w, const int* __restrict__ place,
                                                   const int* __restrict__ rows_end, int64_t tokens, int k, int lanes,
                                                   unsigned cw, Blocks bl, T* __restrict__ g_y,
                                                   row_sum_t<T>* __restrict__ dots) {
  typedef row_vec_t<T, V> Vec;
  typedef row_sum_t<T> S;
  const int64_t s = (int64_t)blockIdx.x * (WG / lanes) + (int)threadIdx.x / lanes, n = tokens * k;
  if (s >= n) return;   // (whole groups of lanes; the shuffles stay inside one)
  const unsigned lane = threadIdx.x % lanes;
  const int64_t t = (uint64_t)s / (unsigned)k;
  const int p = place_of(place, s, n);
  const bool kept = p < *rows_end;
  const S f = w ? w[s] : (S)1;
  S dot = 0;
  for (unsigned c0 = lane; c0 < cw; c0 += U * lanes) {
    Vec xv[U], yv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned c = min(c0 + u * lanes, cw - 1);
      xv[u] = ((const Vec*)x)[bl.at(tokens, t, c)];
      yv[u] = ((const Vec*)y)[bl.at(n, p, c)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned c = c0 + u * lanes;
      if (c >= cw) break;
      S a[V], b[V];
      row_widen<T, V>(xv[u], a);
      row_widen<T, V>(yv[u], b);
#pragma unroll
      for (int i = 0; i < V; ++i) dot += kept ? a[i] * b[i] : (S)0;
      if (g_y) {
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = kept ? f * a[i] : (S)0;
        put<true>((Vec*)g_y + bl.at(n, p, c), row_round<T, V>(a));
      }
    }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
  if (lane == 0) dots[s] = dot;
}

// (a launch holds less than 2^32 threads)
constexpr int64_t MAX_GRID = (1 << 24) - 1;
bool grid_ok(int64_t blocks) { return blocks <= MAX_GRID; }

// the blocks in chunks of V elements; false if a width has a remainder
bool make_blocks(int32_t blocks, const int64_t* widths, int V, Blocks* bl) {
  bl->count = blocks;
  int64_t s = 0;
  for (int b = 0; b <= TACE_ROW_MAX_BLOCKS; ++b) {
    bl->start[b] = (unsigned)(s / V);
    if (b < blocks) {
      if (widths[b] % V) return false;
      s += widths[b];
    }
  }
  return true;
}

const char* route_bad(int type, int64_t tokens, int32_t k, int32_t blocks, const int64_t* widths) {
  if (type < 0 || type > TACE_ROW_F16) return "tace_route: unknown row type";
  if (tokens < 0 || k < 1 || tokens > (INT32_MAX - 8192) / k) return "tace_route: bad sizes";
  if (blocks < 1 || blocks > TACE_ROW_MAX_BLOCKS || !widths) return "tace_route: 1 to 8 blocks";
  int64_t D = 0;
  for (int b = 0; b < blocks; ++b) {
    if (widths[b] < 1 || widths[b] > (1 << 24)) return "tace_route: bad block width";
    D += widths[b];
  }
  if (D > MAX_ROW) return "tace_route: rows of over 32768 elements";
  return nullptr;
}

}  // namespace

extern "C" int tace_rows_abi_version(void) { return TACE_ROWS_ABI_VERSION; }

extern "C" int tace_embed_fwd(int type, int index_bytes, const void* table, const void* tokens, int64_t n,
                              int64_t vocab, int32_t channels, double scale, void* out, void* stream) {
  if (n < 0 || vocab < 0 || vocab > INT32_MAX || channels < 1 || channels > MAX_ROW)
    return tace_fail_msg("tace_embed_fwd: bad sizes");
  if (index_bytes != 4 && index_bytes != 8) return tace_fail_msg("tace_embed_fwd: indices of 4 or 8 bytes");
  if (n == 0) return 0;
  if ((vocab && !table) || !tokens || !out) return tace_fail_msg("tace_embed_fwd: null pointer");
  bool fits = true;
  const bool known = row_dispatch(type, [&](auto z) {
    typedef decltype(z) T;
    row_moves<T>(
        [&](int v, int bytes) { return channels % v == 0 && ((uintptr_t)table | (uintptr_t)out) % bytes == 0; },
        [&](auto vc) {
          constexpr int V = decltype(vc)::value;
          const RowChunks rc{n * (channels / V), row_div((unsigned)(channels / V))};
          const int64_t grid = (rc.total + WG - 1) / WG;
          fits = grid_ok(grid);
          if (!fits) return;
          auto go = [&](auto i) {
            typedef decltype(i) I;
            hipLaunchKernelGGL((k_embed_fwd<T, V, I>), dim3((unsigned)grid), dim3(WG), 0, (hipStream_t)stream,
                               (const T*)table, (const I*)tokens, rc, vocab, (row_sum_t<T>)scale, (T*)out);
          };
          if (index_bytes == 4) go(int32_t());
          else go(int64_t());
        });
  });
  if (!known) return tace_fail_msg("tace_embed_fwd: unknown row type");
  if (!fits) return tace_fail_msg("tace_embed_fwd: too many rows");
  return tace_check_launch("tace_embed_fwd");
}

extern "C" int tace_embed_grad_grouped(int64_t n, int64_t vocab) { return embed_form(n, vocab) == GROUPED; }

extern "C" int64_t tace_embed_grad_work(int type, int64_t n, int64_t vocab, int32_t channels, int grouped) {
  if (n < 1 || vocab < 1 || channels < 1 || channels > MAX_ROW) return 0;
  const int64_t row = (int64_t)channels * (type == TACE_ROW_F64 ? 8 : 4);
  if (!grouped) {
    const int form = embed_form(n, vocab);
    return form == SORTS || form == BUCKETS ? LocalWork(n, vocab, channels, row).bytes : 0;
  }
  // (rows may be moved by 16 bytes, 8, or one element: the largest count of workgroups)
  const int bytes = type == TACE_ROW_F64 ? 8 : type == TACE_ROW_F32 ? 4 : 2;
  int64_t wgs = 0;
  for (int v : {1, 8 / bytes, 16 / bytes})
    if (channels % v == 0) wgs = std::max(wgs, embed_wgs(n, embed_lanes(channels / v)));
  return wgs * 2 * row;
}

extern "C" int tace_embed_grad(int type, int index_bytes, const void* g, const void* tokens, const int32_t* order,
                               const int32_t* rowptr, int64_t n, int64_t vocab, int32_t channels, double scale,
                               void* grad, void* work, int64_t work_bytes, void* stream) {
  if (n < 0 || vocab < 0 || n > INT32_MAX - 8192 || vocab > INT32_MAX - 8192 || channels < 1 || channels > MAX_ROW)
    return tace_fail_msg("tace_embed_grad: bad sizes");
  if (index_bytes != 4 && index_bytes != 8) return tace_fail_msg("tace_embed_grad: indices of 4 or 8 bytes");
  if (type < 0 || type > TACE_ROW_F16) return tace_fail_msg("tace_embed_grad: unknown row type");
  if (vocab == 0) return 0;
  const bool grouped = order != nullptr;
  const int form = grouped ? GROUPED : embed_form(n, vocab);
  if (!grad || (n && (!g || !tokens))) return tace_fail_msg("tace_embed_grad: null pointer");
  if (grouped && n == 0) return tace_fail_msg("tace_embed_grad: no rows, and a grouping of them");
  if (!grouped && form == GROUPED)
    return tace_fail_msg("tace_embed_grad: too many rows and tokens without a grouping");
  if (grouped && !rowptr) return tace_fail_msg("tace_embed_grad: null pointer");
  if (form != SCANS && (!work || work_bytes < tace_embed_grad_work(type, n, vocab, channels, grouped) ||
                        !row_aligned(work)))
    return tace_fail_msg("tace_embed_grad: workspace too small or not 16-byte aligned");
  row_dispatch(type, [&](auto z) {
    typedef decltype(z) T;
    typedef row_sum_t<T> S;
    if (n == 0) {
      const int64_t total = vocab * channels, grid = std::min<int64_t>((total + WG - 1) / WG, 4096);
      hipLaunchKernelGGL((k_embed_grad_none<T>), dim3((unsigned)grid), dim3(WG), 0, (hipStream_t)stream, total,
                         (T*)grad);
      return;
    }
    row_moves<T>(
        [&](int v, int bytes) { return channels % v == 0 && ((uintptr_t)g | (uintptr_t)grad) % bytes == 0; },
        [&](auto vc) {
          constexpr int V = decltype(vc)::value;
          const int cw = channels / V, lanes = embed_lanes(cw), tiles = (cw + lanes - 1) / lanes;
          const int per = embed_per(n, lanes), wgs = (int)embed_wgs(n, lanes), groups = WG / lanes;
          hipStream_t s = (hipStream_t)stream;
          auto go = [&](auto i) {
            typedef decltype(i) I;
            if (form == SCANS) {
              const int ln = std::min(lanes, vocab < 64 ? 8 : 64);
              hipLaunchKernelGGL((k_embed_grad_scan<T, V, I>), dim3((unsigned)vocab, (unsigned)((cw + ln - 1) / ln)),
                                 dim3(WG), 0, s, (const T*)g, (const I*)tokens, (int)n, channels, ln, (S)scale,
                                 (T*)grad);
              return;
            }
            const int columns = (channels + JOIN_COLS - 1) / JOIN_COLS;
            if (form == SORTS || form == BUCKETS) {
              const LocalWork lw(n, vocab, channels, channels * (int64_t)sizeof(S));
              char* at = (char*)work;
              int *bptr = (int*)(at + lw.bptr), *by = (int*)(at + lw.order), *first = (int*)(at + lw.first);
              int* seen = (int*)(at + lw.seen);
              S* sums = (S*)(at + lw.part);
              // (16 threads a row where that leaves the GPU few workgroups)
              const int ln = lw.wgs < 512 && cw > 16 ? 16 : lanes, rows = local_rows(n, channels);
              const dim3 grid((unsigned)lw.wgs, (unsigned)((cw + ln - 1) / ln));
              if (form == SORTS) {
                hipLaunchKernelGGL((k_embed_grad_local<T, V, I, false>), grid, dim3(WG), 0, s, (const T*)g,
                                   (const I*)tokens, nullptr, nullptr, 0, (int)n, (int)vocab, channels, rows, ln,
                                   nullptr, seen, sums);
                hipLaunchKernelGGL((k_embed_grad_total<T, 16, 1>), dim3((unsigned)vocab, (unsigned)columns), dim3(WG),
                                   0, s, seen, nullptr, (int)lw.wgs, (int)vocab, channels, (S)scale, sums, (T*)grad);
                return;
              }
              const int buckets = (int)buckets_of(vocab);
              int few, steps;
              few_fits(n, buckets, &few, &steps);
              few_group((const I*)tokens, 1, (int)n, FewKeys{(int)vocab, BUCKET_BITS, buckets}, few, steps, bptr, by,
                        nullptr, (int32_t*)(at + lw.hist), s);
              hipLaunchKernelGGL((k_embed_grad_local<T, V, I, true>), grid, dim3(WG), 0, s, (const T*)g,
                                 (const I*)tokens, by, bptr, buckets, (int)n, (int)vocab, channels, rows, ln, first,
                                 seen, sums);
              hipLaunchKernelGGL((k_embed_grad_total<T, 32, 2>),
                                 dim3((unsigned)((vocab + 1) / 2), (unsigned)((channels + 31) / 32)), dim3(WG), 0, s,
                                 seen, first, 0, (int)vocab, channels, (S)scale, sums, (T*)grad);
              return;
            }
            hipLaunchKernelGGL((k_embed_grad_part<T, V, I>), dim3((unsigned)wgs, (unsigned)tiles), dim3(WG), 0, s,
                               (const T*)g, (const I*)tokens, order, (int)n, (int)vocab, channels, per, lanes,
                               (S)scale, (T*)grad, (S*)work);
            const int seams = wgs - 1;
            const int64_t zeros = (vocab + 4 * columns - 1) / (4 * columns);
            hipLaunchKernelGGL((k_embed_grad_join<T, I>),
                               dim3((unsigned)(seams + (zeros < 2048 ? zeros : 2048)), (unsigned)columns), dim3(WG), 0,
                               s, (const I*)tokens, order, rowptr, (int)n, (int)vocab, channels,
                               (int64_t)per * groups, seams, (S)scale, (const S*)work, (T*)grad);
          };
          if (index_bytes == 4) go(int32_t());
          else go(int64_t());
        });
  });
  return tace_check_launch("tace_embed_grad");
}

extern "C" int64_t tace_route_group_work(int64_t n, int64_t n_keys) {
  int wgs, steps;
  if (n < 0 || n_keys < 0 || n > INT32_MAX - 8192 || n_keys > INT32_MAX - 8192) return 0;
  if (few_fits(n, n_keys, &wgs, &steps)) return (int64_t)wgs * (n_keys + 1);
  return tace_group_keys_work(n, n_keys) + n;   // (and the keys in 32 bits)
}

extern "C" int tace_route_group(int index_bytes, const void* keys, int64_t stride, int64_t n, int64_t n_keys,
                                int32_t* rowptr, int32_t* order, int32_t* place, int32_t* work, void* stream) {
  if (n < 0 || n_keys < 0 || n > INT32_MAX - 8192 || n_keys > INT32_MAX - 8192)
    return tace_fail_msg("tace_route_group: bad sizes");
  if (index_bytes != 4 && index_bytes != 8) return tace_fail_msg("tace_route_group: indices of 4 or 8 bytes");
  if (!rowptr || !work || (n && (!keys || !order))) return tace_fail_msg("tace_route_group: null pointer");
  hipStream_t s = (hipStream_t)stream;
  int wgs, steps;
  if (few_fits(n, n_keys, &wgs, &steps)) {
    const FewKeys fk{(int)n_keys, 0, (int)n_keys};
    if (index_bytes == 4)
      few_group((const int32_t*)keys, stride, (int)n, fk, wgs, steps, rowptr, order, place, work, s);
    else
      few_group((const int64_t*)keys, stride, (int)n, fk, wgs, steps, rowptr, order, place, work, s);
    return tace_check_launch("tace_route_group");
  }
  int32_t* k32 = work + tace_group_keys_work(n, n_keys);
  const int rc = tace_group_keys(index_bytes, keys, stride, nullptr, n, n_keys, k32, rowptr, order, nullptr, 0, nullptr,
                                 work, nullptr, stream);
  if (rc || !place || n == 0) return rc;
  hipLaunchKernelGGL(k_route_place, dim3((unsigned)((n + WG - 1) / WG)), dim3(WG), 0, s, order, (int)n, place);
  return tace_check_launch("tace_route_group");
}

namespace {

// Rows that go to scattered places are stored past the caches where they are
// whole 128-byte lines (12,288 x 2 rows of 2,048 float32 take 1.16 times as long
// through them), not where two rows meet in a line (20,000 x 4 rows of 400 float16
// take 1.7 times as long past them).
bool whole_lines(int32_t blocks, const int64_t* widths, int size) {
  for (int b = 0; b < blocks; ++b)
    if (widths[b] * size % 128) return false;
  return true;
}

template <typename F>
void route_flag(bool on, F&& f) {
  if (on) f(std::true_type());
  else f(std::false_type());
}

// f(row type, elements a chunk, blocks in chunks, chunks a row); at: the rows'
// addresses, or-ed
template <typename F>
void route_go(int type, int32_t blocks, const int64_t* widths, uintptr_t at, F&& f) {
  row_dispatch(type, [&](auto z) {
    Blocks bl;
    row_moves<decltype(z)>([&](int v, int bytes) { return at % bytes == 0 && make_blocks(blocks, widths, v, &bl); },
                           [&](auto vc) {
                             make_blocks(blocks, widths, decltype(vc)::value, &bl);
                             f(z, vc, bl, bl.start[blocks]);
                           });
  });
}

}  // namespace

extern "C" int tace_route_dispatch(int type, const void* x, const void* weights, const int32_t* place,
                                   const int32_t* rows_end, int64_t tokens, int32_t k, int32_t blocks,
                                   const int64_t* widths, void* out, void* stream) {
  if (const char* bad = route_bad(type, tokens, k, blocks, widths)) return tace_fail_msg(bad);
  if (tokens == 0) return 0;
  if (!x || !place || !rows_end || !out) return tace_fail_msg("tace_route_dispatch: null pointer");
  bool fits = true;
  route_go(type, blocks, widths, (uintptr_t)x | (uintptr_t)out, [&](auto z, auto vc, const Blocks& bl, unsigned cw) {
    typedef decltype(z) T;
    constexpr int V = decltype(vc)::value;
    const RowChunks rc{tokens * cw, row_div(cw)};
    const int64_t grid = (rc.total + WG - 1) / WG;
    fits = grid_ok(grid);
    if (!fits) return;
    route_flag(whole_lines(blocks, widths, sizeof(T)), [&](auto st) {
      hipLaunchKernelGGL((k_route_dispatch<T, V, decltype(st)::value>), dim3((unsigned)grid), dim3(WG), 0,
                         (hipStream_t)stream, (const T*)x, (const row_sum_t<T>*)weights, place, rows_end, rc, tokens, k,
                         bl, (T*)out);
    });
  });
  if (!fits) return tace_fail_msg("tace_route_dispatch: too many rows");
  return tace_check_launch("tace_route_dispatch");
}

extern "C" int tace_route_combine(int type, const void* y, const void* weights, const int32_t* place,
                                  const int32_t* rows_end, int64_t tokens, int32_t k, int32_t blocks,
                                  const int64_t* widths, void* out, void* stream) {
  if (const char* bad = route_bad(type, tokens, k, blocks, widths)) return tace_fail_msg(bad);
  if (tokens == 0) return 0;
  if (!y || !place || !rows_end || !out) return tace_fail_msg("tace_route_combine: null pointer");
  bool fits = true;
  route_go(type, blocks, widths, (uintptr_t)y | (uintptr_t)out, [&](auto z, auto vc, const Blocks& bl, unsigned cw) {
    typedef decltype(z) T;
    constexpr int V = decltype(vc)::value;
    const RowChunks rc{tokens * cw, row_div(cw)};
    const int64_t grid = (rc.total + WG - 1) / WG;
    fits = grid_ok(grid);
    if (!fits) return;
    auto go = [&](auto kc) {
      hipLaunchKernelGGL((k_route_combine<T, V, decltype(kc)::value>), dim3((unsigned)grid), dim3(WG), 0,
                         (hipStream_t)stream, (const T*)y, (const row_sum_t<T>*)weights, place, rows_end, rc, tokens, k,
                         bl, (T*)out);
    };
    if (k == 1) go(std::integral_constant<int, 1>());
    else if (k == 2) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 4>());
  });
  if (!fits) return tace_fail_msg("tace_route_combine: too many rows");
  return tace_check_launch("tace_route_combine");
}

extern "C" int tace_route_dots(int type, const void* x, const void* y, const void* weights, const int32_t* place,
                               const int32_t* rows_end, int64_t tokens, int32_t k, int32_t blocks,
                               const int64_t* widths, void* g_y, void* dots, void* stream) {
  if (const char* bad = route_bad(type, tokens, k, blocks, widths)) return tace_fail_msg(bad);
  if (tokens == 0) return 0;
  if (!x || !y || !place || !rows_end || !dots) return tace_fail_msg("tace_route_dots: null pointer");
  bool fits = true;
  route_go(type, blocks, widths, (uintptr_t)x | (uintptr_t)y | (uintptr_t)g_y,
           [&](auto z, auto vc, const Blocks& bl, unsigned cw) {
             typedef decltype(z) T;
             constexpr int V = decltype(vc)::value;
             int lanes = 1;
             while (lanes < 64 && (unsigned)lanes < cw) lanes *= 2;
             const int64_t groups = WG / lanes, grid = (tokens * k + groups - 1) / groups;
             fits = grid_ok(grid);
             if (!fits) return;
             auto go = [&](auto uc) {
               hipLaunchKernelGGL((k_route_dots<T, V, decltype(uc)::value>), dim3((unsigned)grid), dim3(WG), 0,
                                  (hipStream_t)stream, (const T*)x, (const T*)y, (const row_sum_t<T>*)weights, place,
                                  rows_end, tokens, k, lanes, cw, bl, (T*)g_y, (row_sum_t<T>*)dots);
             };
             if (cw <= (unsigned)lanes) go(std::integral_constant<int, 1>());
             else if (cw <= 2u * lanes) go(std::integral_constant<int, 2>());
             else go(std::integral_constant<int, 4>());
           });
  if (!fits) return tace_fail_msg("tace_route_dots: too many rows");
  return tace_check_launch("tace_route_dots");
}
