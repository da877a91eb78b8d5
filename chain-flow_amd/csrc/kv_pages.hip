// The pages of the paged key / value cache on MI355X: accepted rows moved together, pages shared between sequences, taken
// and given back.  A pool's book-keeping is three tensors: table [S][W] (the pages of each sequence, -1: none), room [S]
// (tokens that a sequence's pages are for: it holds ceil(room / page) of them) and ref [blocks] (sequences that hold a page;
// 0: free).  Everything is decided on the device, in an order that the sequences give (the lowest free page first), so
// that a call never synchronises, can be captured, and gives the same table every time.
#include <algorithm>
#include <type_traits>

#include "cfh_host.h"
#include "cfh_scan.h"

namespace {

typedef unsigned v4u __attribute__((ext_vector_type(4)));   // (arrays of uint4, a union, go to memory)

// One part of the cache (keys, values) of all layers, in bytes.
struct Part { char* p; uint8_t* ex; long long ls, bs, es; };   // base, scale bytes, strides of a layer, a block, a layer's scales

struct PoolArgs {
  Part part[2];
  int layers, blocks, page, Hkv;
  int row;                   // bytes of a token's heads
  bool f8;
};

// Keys (0) or values (1), field by field: the array taken by a lane's index would go to memory.
__device__ __forceinline__ Part part_of(const PoolArgs& c, int i) {
  const Part &k = c.part[0], &v = c.part[1];
  return {i ? v.p : k.p, i ? v.ex : k.ex, i ? v.ls : k.ls, i ? v.bs : k.bs, i ? v.es : k.es};
}

// ---------------------------------------------------------------------------- accepted rows
// Node path[s][i] of sequence s, row lens[s] + path[s][i], becomes row lens[s] + i, in every layer.  The nodes ascend, so
// row i never lies behind its source and no source lies before the row in hand: a thread that moves one 16-byte column
// of all rows in order, whole batches read before they are written, needs no other thread.  Bound by round trips (lengths, path
// and table, rows), not bytes: one path in 8 layers of 4 x 256 bf16 4.9 us, 48 in 16 layers of 2 x 128 e4m3 (2.5 MB) 5.8.
struct CommitArgs {
  PoolArgs c;
  const int* table;          // [S][table_ld]
  const int* lens;           // [S]
  const int* path;           // [S][path_ld]
  const int* count;          // [S]
  int* status;
  int table_ld, W, path_ld, most;
};

constexpr int COMMIT_ROWS = 64;   // path entries whose slots lie in LDS at a time
constexpr int COMMIT_BATCH = 8;   // rows a thread has in flight

__global__ void __launch_bounds__(256) k_commit(CommitArgs a) {
  __shared__ int src[COMMIT_ROWS], dst[COMMIT_ROWS];
  __shared__ int bad;
  const int s = blockIdx.y, n = a.count[s], len = a.lens[s];
  if (n <= 0) return;                                // nothing accepted, or padding
  const int* path = a.path + (size_t)s * a.path_ld;
  const int* table = a.table + (size_t)s * a.table_ld;
  // the whole path first: ascending nodes whose rows the table holds
  if (threadIdx.x == 0) bad = n > a.most || len < 0;
  __syncthreads();
  const long long limit = (long long)a.W * a.c.page;
  auto slot_of = [&](long long pos) __attribute__((always_inline)) {                // -1: not in the cache
    const int blk = pos < limit ? table[pos / a.c.page] : -1;
    return blk < 0 || blk >= a.c.blocks ? -1 : blk * a.c.page + (int)(pos % a.c.page);
  };
  if (!bad)
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int p = path[i], from = slot_of((long long)len + max(p, 0)), to = slot_of((long long)len + i);
      if (p < (i ? path[i - 1] + 1 : 0) || from < 0 || to < 0) bad = 1;
      if (i < COMMIT_ROWS) { src[i] = from; dst[i] = to; }
    }
  __syncthreads();
  if (bad) {
    if (threadIdx.x == 0 && a.status) a.status[0] = 1;
    return;
  }
  const int cols = a.c.row / 16, per = cols + (a.c.f8 ? a.c.Hkv : 0);
  const int item = blockIdx.x * blockDim.x + threadIdx.x, unit = item / per, col = item - unit * per;
  const bool live = unit < 2 * a.c.layers;
  const Part q = part_of(a.c, unit & 1);
  const size_t layer = live ? unit >> 1 : 0;
  for (int i0 = 0; i0 < n; i0 += COMMIT_ROWS) {
    const int m = min(COMMIT_ROWS, n - i0);
    if (i0) {
      __syncthreads();
      if (threadIdx.x < m) {
        src[threadIdx.x] = slot_of((long long)len + path[i0 + threadIdx.x]);
        dst[threadIdx.x] = slot_of((long long)len + i0 + threadIdx.x);
      }
      __syncthreads();
    }
    if (!live) continue;
    for (int i = 0; i < m; i += COMMIT_BATCH) {
      if (col < cols) {
        v4u x[COMMIT_BATCH];
        auto at = [&](int slot) __attribute__((always_inline)) {
          return (v4u*)(q.p + layer * q.ls + (size_t)(slot / a.c.page) * q.bs + (size_t)(slot % a.c.page) * a.c.row) + col;
        };
#pragma unroll
        for (int u = 0; u < COMMIT_BATCH; ++u) x[u] = *at(src[min(i + u, m - 1)]);
#pragma unroll
        for (int u = 0; u < COMMIT_BATCH; ++u)
          if (i + u < m) *at(dst[i + u]) = x[u];
      } else {
        uint8_t x[COMMIT_BATCH];
        auto at = [&](int slot) __attribute__((always_inline)) { return q.ex + layer * q.es + (size_t)slot * a.c.Hkv + (col - cols); };
#pragma unroll
        for (int u = 0; u < COMMIT_BATCH; ++u) x[u] = *at(src[min(i + u, m - 1)]);
#pragma unroll
        for (int u = 0; u < COMMIT_BATCH; ++u)
          if (i + u < m) *at(dst[i + u]) = x[u];
      }
    }
  }
}

// ---------------------------------------------------------------------------- fork
// Row dst[i] of the table lets go of its pages and shares row src[i]'s (src -1: none).  No source is a destination
// of another pair and destinations differ (pairs that break this are skipped), so that pairs need no order; holders
// are counted by atomic additions, whose order does not matter.  A workgroup a pair, two round trips through the table: 30,011
// tokens' 469 pages shared by 8 sequences 5.4 us, 24 prompts of 13 pages by 4 each 4.2.
struct ForkArgs {
  int* table;
  int* room;
  int* ref;
  const int* src;            // [n]
  const int* dst;
  int* status;
  int table_ld, W, S, blocks, page, n;
};

__global__ void __launch_bounds__(256) k_fork(ForkArgs a) {
  __shared__ int clash;
  const int i = blockIdx.x, t = threadIdx.x, from = a.src[i], to = a.dst[i];
  if (to == -1) return;                              // padding
  if (t == 0) clash = 0;
  __syncthreads();
  for (int j = t; j < a.n; j += blockDim.x)
    if (j != i && (a.dst[j] == to || (from >= 0 && a.dst[j] == from))) clash = 1;
  __syncthreads();
  const long long limit = (long long)a.W * a.page;
  const bool in = to >= 0 && to < a.S && from >= -1 && from < a.S;
  const int had_room = in ? a.room[to] : -1, new_room = in ? (from >= 0 ? a.room[from] : 0) : -1;
  if (clash || had_room < 0 || new_room < 0 || had_room > limit || new_room > limit) {
    if (t == 0 && a.status) a.status[0] = 1;
    return;
  }
  if (from == to) return;
  int* row = a.table + (size_t)to * a.table_ld;
  const int* other = a.table + (size_t)max(from, 0) * a.table_ld;
  const int had = (int)(((long long)had_room + a.page - 1) / a.page), want = (int)(((long long)new_room + a.page - 1) / a.page);
  for (int j = t; j < max(had, want); j += blockDim.x) {
    int now = -1;
    if (j < had) {
      const int p = row[j];
      if (p >= 0 && p < a.blocks) atomicSub(&a.ref[p], 1);
      else if (a.status) a.status[0] = 1;
    }
    if (j < want) {
      now = other[j];
      if (now >= 0 && now < a.blocks) atomicAdd(&a.ref[now], 1);
      else if (a.status) a.status[0] = 1;
    }
    row[j] = now;
  }
  __syncthreads();
  if (t == 0) a.room[to] = new_room;
}

// ---------------------------------------------------------------------------- resize
struct ResizeArgs {
  PoolArgs c;
  int* table;
  int* room;
  int* ref;
  const int* new_room;
  int* status;
  int4* plan;                // [S]: first place in `fresh` (-1: refused), page to copy (-1: none), pages kept, tokens in the copied one
  int4* copies;              // [S + 1]: how many pages are copied (x of the first), then from, to, tokens of each
  int* fresh;                // pages taken, in order
  int table_ld, W, S, pieces;
};

constexpr int RS_MAX = 4096;      // sequences of a call
constexpr int RS_T = 1024;
constexpr int RS_FAR = 0x3fffffff; // a place behind every page
// Up to so many table entries (and RS_T sequences) one workgroup does all of it, in one launch; above, the entries are let go of
// and filled in by a workgroup a sequence, in launches before and behind.  A pair of calls that grows and shrinks 48
// sequences of 567 entries: 14.8 us so, 25.3 in three launches each (200 of 304: 15.7, 26.5; 1,000 of 223: 19.9, 26.4); a pair in
// which every page changes hands 41 and 34 (79 and 41; 266 and 89).  The cost goes with the pages that change, which the host does not
// know: the rule takes the side of growing by a step's rows and back, which every step does, and loses where prompts come and go.
constexpr long long RS_ONE = 65536;

// Pages that a sequence has, wants and keeps.
struct Span { int had, want, kept, part; bool ok, pad; };
__device__ __forceinline__ Span span_of(const ResizeArgs& a, int s) {
  const long long limit = (long long)a.W * a.c.page;
  const int now = a.room[s], want = a.new_room[s];
  Span x = {};
  x.pad = want < 0;
  x.ok = !x.pad && now >= 0 && now <= limit && want <= limit;
  if (x.ok) {
    x.had = (int)(((long long)now + a.c.page - 1) / a.c.page);
    x.want = (int)(((long long)want + a.c.page - 1) / a.c.page);
    x.kept = min(x.had, x.want);
    x.part = want > now ? now % a.c.page : 0;
  }
  return x;
}

// An entry behind its sequence's new room: the page has one holder less.
__device__ __forceinline__ void let_go(const ResizeArgs& a, int s, int j) {
  int* entry = a.table + (size_t)s * a.table_ld + j;
  const int p = *entry;
  if (p >= 0 && p < a.c.blocks) atomicSub(&a.ref[p], 1);
  else if (a.status) a.status[0] = 1;
  *entry = -1;
}

// First: pages behind the new rooms are let go of.
__global__ void __launch_bounds__(64) k_release(ResizeArgs a) {
  const int s = blockIdx.x;
  const Span x = span_of(a, s);
  if (!x.ok) {
    if (!x.pad && threadIdx.x == 0 && a.status) a.status[0] = 1;
    return;
  }
  for (int j = x.want + (int)threadIdx.x; j < x.had; j += 64) let_go(a, s, j);
}

// The sum of v over the threads before this one, and over all of them.
template <typename N>
__device__ __forceinline__ N scan_before(N v, N* tmp, N& all) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const N run = scan64(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = run;
  __syncthreads();
  N before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < RS_T / 64; ++w) {
    if (w < wave) before += tmp[w];
    all += tmp[w];
  }
  return before + run - v;
}

// The last i in [0, n) with first[i] <= v (first[0] = 0, ascending).
__device__ __forceinline__ int last_at(const int* first, int n, int v) {
  int lo = 0;
  for (int step = RS_T / 2; step; step /= 2)
    if (lo + step < n && first[lo + step] <= v) lo += step;
  return lo;
}

// The growing sequences that share a last page: their number, and the last of them, in a table of the pages by open addressing
// (counts and a maximum: the order of the additions does not matter; twice as many entries as sequences).  4,000
// sequences that grow out of one page: 100 us of growing, 260 with each against each.
template <int SIZE>
struct Shared {
  int page[SIZE], count[SIZE], last[SIZE];
  __device__ void clear() {
    for (int i = threadIdx.x; i < SIZE; i += RS_T) { page[i] = -1; count[i] = 0; last[i] = -1; }
  }
  __device__ int place(int p) {
    unsigned i = (unsigned)p * 2654435761u % SIZE;
    for (int tries = 0; tries < SIZE; ++tries, i = (i + 1) % SIZE) {
      const int was = atomicCAS(&page[i], -1, p);
      if (was == -1 || was == p) break;
    }
    return (int)i;
  }
};

// Then, in one workgroup, as every place depends on those before it: what each sequence needs, in order, and the lowest free pages for it.  A shared last page
// that is filled in part is copied before its sequence grows: by all but the last of its holders.  ONE: letting go and filling in,
// too.
template <bool ONE>
__global__ void __launch_bounds__(RS_T) k_plan(ResizeArgs a) {
  constexpr int MOST = ONE ? RS_T : RS_MAX;
  __shared__ int tails[MOST];        // the shared page a sequence would write into, -1: none
  __shared__ Shared<2 * MOST> shared;
  // ONE: a sequence a thread, what others need of it in LDS, as are the first pages taken (a pair of calls for 48 sequences in a
  // graph: 18.4 us, 20.0 through memory; 96 copied pages: this kernel 10.4 for 12.0)
  constexpr int QUICK = ONE ? 4096 : 1;
  __shared__ int first[ONE ? RS_T : 1], quick[QUICK];
  __shared__ int4 plans[ONE ? RS_T : 1];
  __shared__ double tmp[RS_T / 64];
  __shared__ int used, copied_n;
  const int t = threadIdx.x;
  if (t == 0) used = copied_n = 0;
  Span mine = {};
  if (ONE && t < a.S) mine = span_of(a, t);
  auto span = [&](int s) __attribute__((always_inline)) { return ONE ? mine : span_of(a, s); };
  auto plan = [&](int s) __attribute__((always_inline)) -> int4& {
    if constexpr (ONE) return plans[s];
    else return a.plan[s];
  };
  auto fresh = [&](int i) __attribute__((always_inline)) { return i < QUICK && ONE ? quick[i] : a.fresh[i]; };
  if constexpr (ONE) {
    const Span x = mine;
    if (t < a.S && !x.ok && !x.pad && a.status) a.status[0] = 1;
    double all;
    const double at = scan_before((double)(x.ok ? x.had - x.kept : 0), tmp, all);
    const int n = (int)all;                          // (at most RS_ONE entries)
    first[t] = (int)at;
    tails[t] = x.want;
    __syncthreads();
    for (int i0 = t; i0 < n; i0 += 4 * RS_T)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * RS_T;
        if (i >= n) break;
        const int s = last_at(first, a.S, i);
        let_go(a, s, tails[s] + i - first[s]);
      }
    __syncthreads();
  }
  bool any = false;
  for (int s = t; s < a.S; s += RS_T) {
    const Span x = span(s);
    int tail = -1;
    if (x.ok && x.part) {
      tail = a.table[(size_t)s * a.table_ld + x.kept - 1];
      if (tail < 0 || tail >= a.c.blocks) {
        if (a.status) a.status[0] = 1;
        tail = -2;                                   // no such page: refused
      } else if (a.ref[tail] <= 1) {
        tail = -1;
      }
    }
    tails[s] = tail;
    any |= tail >= 0;
  }
  if (__syncthreads_or(any)) {
    shared.clear();
    __syncthreads();
    for (int s = t; s < a.S; s += RS_T)
      if (tails[s] >= 0) {
        const int i = shared.place(tails[s]);
        atomicAdd(&shared.count[i], 1);
        atomicMax(&shared.last[i], s);
      }
    __syncthreads();
  }
  double total = 0;                                  // (what is asked for may pass 32 bits; what is free does not)
  for (int s0 = 0; s0 < a.S; s0 += RS_T) {
    const int s = s0 + t;
    int need = 0, tail = -1;
    Span x = {};
    if (s < a.S) {
      x = span(s);
      tail = tails[s];
      if (tail == -2) x.ok = false;
      if (x.ok) need = x.want - x.kept;
      if (x.ok && tail >= 0) {
        const int i = shared.place(tail);
        if (shared.count[i] < a.ref[tail] || shared.last[i] != s) ++need;
      }
    }
    double all;
    const int at = (int)fmin(total + scan_before((double)need, tmp, all), (double)RS_FAR);
    if (s < a.S) {
      const bool copied = x.ok && need > x.want - x.kept;
      // (-2: keeps its shared page, if those before it copied it)
      plan(s) = make_int4(x.ok ? at : -1, copied ? tail : x.ok && tail >= 0 ? -2 : -1, x.kept, x.part);
    }
    if constexpr (ONE) first[t] = at;
    total += all;
  }
  // The lowest free pages, 16 counts a thread and step: four quarters of a step, four counts of each (whole lines a wave), their
  // sums side by side in one word.  16,384 pages that are taken cost 1.1 us (with 16 counts side by side a thread 1.5).
  constexpr int Q = 4 * RS_T;                        // pages of a quarter
  double base = 0;
  for (int p0 = 0; p0 < a.c.blocks && base < total; p0 += 4 * Q) {
    int ref[16];
    unsigned long long n = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = p0 + q * Q + 4 * t;
      if (at + 4 <= a.c.blocks) {
        __builtin_memcpy(ref + 4 * q, a.ref + at, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) ref[4 * q + e] = at + e < a.c.blocks ? a.ref[at + e] : 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) n += (unsigned long long)(ref[i] == 0) << (i / 4 * 16);
    if (p0 && !__syncthreads_or(n != 0)) continue;
    unsigned long long all;
    unsigned long long before = scan_before(n, (unsigned long long*)tmp, all);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      int to = (int)base + (int)(before >> (16 * q) & 0xffff);   // (below 2^30: so many pages at most)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ref[4 * q + e] == 0) {
          if (to < total) {
            const int page = p0 + q * Q + 4 * t + e;
            if (ONE && to < QUICK) quick[to] = page;
            else a.fresh[to] = page;
          }
          ++to;
        }
      base += (double)(all >> (16 * q) & 0xffff);
    }
  }
  const int have = (int)fmin(base, total);
  __syncthreads();
  for (int s = t; s < a.S; s += RS_T) {
    const int4 p = plan(s);
    if (p.x < 0) continue;
    const Span x = span(s);
    const int need = x.want - x.kept + (p.y >= 0);
    if ((need > 0 || p.y == -2) && p.x + need > have) {
      plan(s).x = -1;
      if (a.status) a.status[0] = 1;
      continue;
    }
    if (p.y >= 0) {
      atomicSub(&a.ref[p.y], 1);
      a.copies[1 + atomicAdd(&copied_n, 1)] = make_int4(p.y, fresh(p.x), p.w, 0);   // (in any order)
    }
    if (need > 0) atomicMax(&used, p.x + need);
    if constexpr (ONE) a.room[s] = a.new_room[s];
  }
  __syncthreads();
  if (t == 0) a.copies[0].x = copied_n;
  for (int i = t; i < used; i += RS_T) {             // (what is used was had: no place behind)
    const int page = fresh(i);
    a.ref[page] = 1;
    if constexpr (ONE) {
      const int s = last_at(first, a.S, i);
      const int4 p = plans[s];
      a.table[(size_t)s * a.table_ld + p.z - (p.y >= 0) + i - p.x] = page;
    }
  }
}

// The tables and rooms, where they are not filled in above.
__global__ void __launch_bounds__(64) k_fill(ResizeArgs a) {
  const int s = blockIdx.x, t = threadIdx.x;
  const int4 p = a.plan[s];
  if (p.x < 0) return;
  const int want = (int)(((long long)a.new_room[s] + a.c.page - 1) / a.c.page), j0 = p.z - (p.y >= 0);
  for (int j = j0 + t; j < want; j += 64) a.table[(size_t)s * a.table_ld + j] = a.fresh[p.x + j - j0];
  if (t == 0) a.room[s] = a.new_room[s];
}

// Last, the copies: a piece of a page of one layer's keys or values at a time.  96 pages in 8 layers (29 of their 64 rows of 4 x 256
// bf16 on average: 180 MB in and out) 41 us, 4.4 TB/s, with the pages in memory; 27 over one pool again and again.  At most 4,096 workgroups, as the number of copies is known here only:
// the whole call and a plan without copies take 55.3 and 6.9 us, with 1,024 of them 56.1 and 6.6, with 16,384 54.3 and 9.2.
constexpr int PIECE = 16384;

__global__ void __launch_bounds__(256) k_copy(ResizeArgs a) {
  const int t = threadIdx.x, units = 2 * a.c.layers * a.pieces;
  const long long all = (long long)a.copies[0].x * units;
  for (long long item = blockIdx.x; item < all; item += gridDim.x) {
    const int4 p = a.copies[1 + item / units];
    const int rest = (int)(item % units), unit = rest / a.pieces, piece = rest % a.pieces;
    const Part q = part_of(a.c, unit & 1);
    const size_t layer = unit >> 1;
    const int bytes = p.z * a.c.row, end = min(bytes, (piece + 1) * PIECE);
    const char* src = q.p + layer * q.ls + (size_t)p.x * q.bs;
    char* dst = q.p + layer * q.ls + (size_t)p.y * q.bs;
    if (piece * PIECE >= bytes) continue;
    constexpr int N = PIECE / (256 * 16);
    v4u x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = *(const v4u*)(src + min(piece * PIECE + (i * 256 + t) * 16, end - 16));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = piece * PIECE + (i * 256 + t) * 16;
      if (o < end) *(v4u*)(dst + o) = x[i];
    }
    if (a.c.f8 && piece == 0) {
      const size_t per = (size_t)a.c.page * a.c.Hkv;
      const uint8_t* es = q.ex + layer * q.es + p.x * per;
      uint8_t* ed = q.ex + layer * q.es + p.y * per;
      for (int o = t; o < p.z * a.c.Hkv; o += 256) ed[o] = es[o];
    }
  }
}

constexpr long long PAGE_MOST = 0x40000000ll - PIECE;   // elements of a page: its last piece ends within 32 bits

int pool_of(const cfh_kv_pool* c, PoolArgs& a) {
  if (!c || c->layers < 1 || c->blocks < 1 || c->page < 1 || c->heads < 1) return CFH_E_INVALID;
  if ((c->dim != 64 && c->dim != 128 && c->dim != 256) || (long long)c->blocks * c->page > 0x7fffffffll ||
      (long long)c->page * c->heads * c->dim > PAGE_MOST)
    return CFH_E_UNSUPPORTED;
  const bool f8 = c->k_exp || c->v_exp;
  const int es = f8 ? 1 : 2;
  const long long inner = (long long)c->page * c->heads * c->dim, scales = (long long)c->blocks * c->page * c->heads;
  if (!c->k || !c->v || (f8 && (!c->k_exp || !c->v_exp)) || ((uintptr_t)c->k | (uintptr_t)c->v) % 16) return CFH_E_INVALID;
  const void* base[2] = {c->k, c->v};
  uint8_t* ex[2] = {c->k_exp, c->v_exp};
  const long long ls[2] = {c->ls_k, c->ls_v}, bs[2] = {c->bs_k, c->bs_v}, xs[2] = {c->ls_k_exp, c->ls_v_exp};
  for (int i = 0; i < 2; ++i) {
    if (bs[i] < inner || bs[i] % 16) return CFH_E_INVALID;
    // layers around the blocks, or blocks around the layers
    if (c->layers > 1 && (ls[i] < inner || ls[i] % 16 || (ls[i] < (c->blocks - 1) * bs[i] + inner && bs[i] < (c->layers - 1) * ls[i] + inner) ||
                          (f8 && xs[i] < scales)))
      return CFH_E_INVALID;
    a.part[i] = {(char*)base[i], ex[i], ls[i] * es, bs[i] * es, xs[i]};
  }
  a.layers = c->layers; a.blocks = c->blocks; a.page = c->page; a.Hkv = c->heads; a.row = c->heads * c->dim * es; a.f8 = f8;
  return CFH_OK;
}

}  // namespace

extern "C" {

int cfh_kv_commit(const cfh_kv_pool* pool, const int32_t* table, int table_ld, int max_blocks, const int32_t* seq_lens,
                  const int32_t* path, int path_ld, int max_path, const int32_t* path_len, int S, int32_t* status,
                  void* stream) {
  CommitArgs a = {};
  if (int rc = pool_of(pool, a.c)) return rc;
  if (S < 0 || max_path < 0 || max_blocks < 0) return CFH_E_INVALID;
  if (S == 0 || max_path == 0) return CFH_OK;
  if (!table || !seq_lens || !path || !path_len || table_ld < max_blocks || path_ld < max_path) return CFH_E_INVALID;
  if (S > 65535) return CFH_E_UNSUPPORTED;
  a.table = table; a.lens = seq_lens; a.path = path; a.count = path_len; a.status = status;
  a.table_ld = table_ld; a.W = max_blocks; a.path_ld = path_ld; a.most = max_path;
  const long long items = 2ll * a.c.layers * (a.c.row / 16 + (a.c.f8 ? a.c.Hkv : 0));
  if (items > 0x3fffffffll) return CFH_E_UNSUPPORTED;
  hipLaunchKernelGGL(k_commit, dim3((unsigned)((items + 255) / 256), S), dim3(256), 0, (hipStream_t)stream, a);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int cfh_kv_fork(int32_t* table, int table_ld, int max_blocks, int32_t* room, int S, int32_t* ref, int blocks, int page,
                const int32_t* src, const int32_t* dst, int n, int32_t* status, void* stream) {
  if (n < 0 || S < 0 || blocks < 1 || page < 1 || max_blocks < 0 || table_ld < max_blocks) return CFH_E_INVALID;
  if (max_blocks > RS_FAR || (long long)max_blocks * page > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  if (n == 0) return CFH_OK;
  if (!table || !room || !ref || !src || !dst) return CFH_E_INVALID;
  if (n > 65535) return CFH_E_UNSUPPORTED;
  ForkArgs a = {table, room, ref, src, dst, status, table_ld, max_blocks, S, blocks, page, n};
  hipLaunchKernelGGL(k_fork, dim3(n), dim3(256), 0, (hipStream_t)stream, a);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

int64_t cfh_kv_resize_ws_bytes(int S, int max_blocks, int blocks) {
  if (S < 0 || max_blocks < 0 || blocks < 1) return -1;
  return 16ll * S + 16 * (S + 1ll) + 4 * std::min((long long)blocks, (long long)S * max_blocks);
}

int cfh_kv_resize(const cfh_kv_pool* pool, int32_t* table, int table_ld, int max_blocks, int32_t* room, int S, int32_t* ref,
                  int blocks, int page, const int32_t* new_room, void* ws, int32_t* status, void* stream) {
  ResizeArgs a = {};
  if (pool) {
    if (int rc = pool_of(pool, a.c)) return rc;
    if (a.c.blocks != blocks || a.c.page != page) return CFH_E_INVALID;
  }
  if (S < 0 || blocks < 1 || page < 1 || max_blocks < 0 || table_ld < max_blocks) return CFH_E_INVALID;
  if (S == 0) return CFH_OK;
  if (!table || !room || !ref || !new_room || !ws || (uintptr_t)ws % 16) return CFH_E_INVALID;
  if (S > RS_MAX || max_blocks > RS_FAR || blocks > RS_FAR || (long long)max_blocks * page > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  a.c.blocks = blocks; a.c.page = page;
  a.table = table; a.room = room; a.ref = ref; a.new_room = new_room; a.status = status;
  a.plan = (int4*)ws; a.copies = a.plan + S; a.fresh = (int*)(a.copies + S + 1);
  a.table_ld = table_ld; a.W = max_blocks; a.S = S;
  a.pieces = pool ? (int)(((long long)page * a.c.row + PIECE - 1) / PIECE) : 0;
  if (2ll * a.c.layers * a.pieces > 0x7fffffffll) return CFH_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (S <= RS_T && (long long)S * max_blocks <= RS_ONE) {
    hipLaunchKernelGGL(k_plan<true>, dim3(1), dim3(RS_T), 0, st, a);
    CFH_LAUNCH_CHECK();
  } else {
    hipLaunchKernelGGL(k_release, dim3(S), dim3(64), 0, st, a);
    CFH_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_plan<false>, dim3(1), dim3(RS_T), 0, st, a);
    CFH_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_fill, dim3(S), dim3(64), 0, st, a);
    CFH_LAUNCH_CHECK();
  }
  if (!pool) return CFH_OK;
  const long long items = 2ll * S * a.c.layers * a.pieces;
  hipLaunchKernelGGL(k_copy, dim3((unsigned)std::min(items, 4096ll)), dim3(256), 0, st, a);
  CFH_LAUNCH_CHECK();
  return CFH_OK;
}

}  // extern "C"
