// Products with a selection matrix that is never written out: the embedding lookup
// (Y = alpha S W + beta Y, S one-hot rows given by token ids), its gradient
// (dW = alpha S^T G + beta dW), and the routing of tokens to experts and back (S has k entries a
// row).  All of them move rows of `dim` values and do one multiply-add a value at most (0.25 to 0.5
// flop a byte): memory bounds them, and on short lists latency does.  A warp takes a slab of the
// columns of a row at a time, so that every load and store of a warp is one contiguous piece of a
// row.  Rates below are the bytes that a call cannot do without per time, on one B200 whose copy
// rate is 6.55 TB/s.
#include <algorithm>

#include "b2s_sort.cuh"

namespace b2s {

constexpr int kSelWarps = 8;            // warps per CTA of the row kernels
constexpr int kSelThreads = 32 * kSelWarps;
constexpr int kSelCols = 256;           // columns of a row a warp holds at a time (8 per lane)
constexpr int64_t kSelMaxDim = 1 << 22; // columns are 32-bit numbers, and slabs few

template <class T> struct acc_of { using type = float; };
template <> struct acc_of<double> { using type = double; };

template <int VB> struct raw_of;
template <> struct raw_of<1> { using type = uint8_t; };
template <> struct raw_of<2> { using type = uint16_t; };
template <> struct raw_of<4> { using type = uint32_t; };
template <> struct raw_of<8> { using type = unsigned long long; };
template <> struct raw_of<16> { using type = uint4; };

// A lane's E columns of a slab of 32 E columns of one row, as U groups of VE neighbouring elements:
// group u begins at column (u * 32 + lane) * VE of the slab.  VE is 16 bytes of the value type
// when bases, pitches and width allow it (a float row beside 16-bit values is then taken in two
// pieces of 16 bytes), else one element; either way the accesses of a warp cover one contiguous
// piece of the row.
template <class O, int VE, int E = 8> struct Part {
  static constexpr int U = E / VE;
  static constexpr int OB = VE == 1 ? static_cast<int>(sizeof(O)) : 16;
  static constexpr int OE = OB / static_cast<int>(sizeof(O));
  static constexpr int N = VE / OE;
  using Raw = typename raw_of<OB>::type;
  Raw r[U * N];

  __device__ static int column(int col0, int u) {
    return col0 + (u * 32 + static_cast<int>(threadIdx.x & 31)) * VE;
  }
  __device__ void load(const O* row, int col0, int dim) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = column(col0, u);
#pragma unroll
      for (int p = 0; p < N; ++p)
        if (c < dim) r[u * N + p] = *reinterpret_cast<const Raw*>(row + c + p * OE);
    }
  }
  __device__ void store(O* row, int col0, int dim) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = column(col0, u);
#pragma unroll
      for (int p = 0; p < N; ++p)
        if (c < dim) *reinterpret_cast<Raw*>(row + c + p * OE) = r[u * N + p];
    }
  }
  __device__ typename acc_of<O>::type get(int i) const {
    O v;
    memcpy(&v, reinterpret_cast<const char*>(r) + i * sizeof(O), sizeof(O));
    return to_acc(v);
  }
  // elements 2 i and 2 i + 1, for sums in pairs
  __device__ float2 pair(int i) const {
    if constexpr (VE > 1 && sizeof(O) == 2) {
      uint32_t w;
      memcpy(&w, reinterpret_cast<const char*>(r) + 4 * i, 4);
      if constexpr (std::is_same_v<O, bf16>)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
      __half2 h;
      memcpy(&h, &w, 4);
      return __half22float2(h);
    } else {
      return make_float2(get(2 * i), get(2 * i + 1));
    }
  }
  __device__ void set(int i, typename acc_of<O>::type a) {
    const O v = storage_of<O>::from_acc(a);
    memcpy(reinterpret_cast<char*>(r) + i * sizeof(O), &v, sizeof(O));
  }
};

// E sums beside a Part: float32 ones are kept and added in pairs (one instruction for two)
template <class A, int E> struct Sums {
  A v[E];
  __device__ void clear() {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = A(0);
  }
  template <class P> __device__ void set(const P& p) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = p.get(e);
  }
  template <class P> __device__ void add(const P& p) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] + p.get(e);
  }
  template <class P> __device__ void fma(A w, const P& p) {
#pragma unroll
    for (int e = 0; e < E; ++e) fma_acc(v[e], w, p.get(e));
  }
};
template <int E> struct Sums<float, E> {
  float2 v2[E / 2];
  __device__ void clear() {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v2[e] = make_float2(0.f, 0.f);
  }
  template <class P> __device__ void set(const P& p) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v2[e] = p.pair(e);
  }
  template <class P> __device__ void add(const P& p) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v2[e] = __fadd2_rn(v2[e], p.pair(e));
  }
  template <class P> __device__ void fma(float w, const P& p) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) v2[e] = __ffma2_rn(make_float2(w, w), p.pair(e), v2[e]);
  }
};
template <class A, int E> __device__ inline A sum_of(const Sums<A, E>& s, int e) {
  if constexpr (std::is_same_v<A, float>)
    return e & 1 ? s.v2[e / 2].y : s.v2[e / 2].x;
  else
    return s.v[e];
}

// sums as they are, stored as O
template <class O, int VE, class A, int E>
__device__ inline void store_sums(O* row, int col0, int dim, const Sums<A, E>& s) {
  Part<O, VE, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) v.set(e, sum_of(s, e));
  v.store(row, col0, dim);
}
// alpha * sums (+ beta * old)
template <class O, int VE, class A, int E>
__device__ inline void store_axpby(O* row, int col0, int dim, const Sums<A, E>& s, A alpha,
                                   bool has_beta, A beta, const Part<O, VE, E>& old) {
  Part<O, VE, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    A x = alpha * sum_of(s, e);
    if (has_beta) x = x + beta * old.get(e);
    v.set(e, x);
  }
  v.store(row, col0, dim);
}
template <class O, int VE, class A, int E>
__device__ inline void store_axpby(O* row, int col0, int dim, const Sums<A, E>& s, A alpha,
                                   bool has_beta, A beta) {
  Part<O, VE, E> old;
  if (has_beta) old.load(row, col0, dim);
  store_axpby<O, VE, A, E>(row, col0, dim, s, alpha, has_beta, beta, old);
}
// a row of zeros: 16 bytes at a time between the first and the last 16-byte border in it
template <class O> __device__ inline void zero_row(O* row, int dim) {
  constexpr int V = 16 / static_cast<int>(sizeof(O));
  const int lane = threadIdx.x & 31;
  O zero;
  memset(&zero, 0, sizeof(O));
  int head = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) /
             static_cast<int>(sizeof(O));
  head = head < dim ? head : dim;
  if (lane < head) row[lane] = zero;
  uint4* body = reinterpret_cast<uint4*>(row + head);
  const int full = (dim - head) / V;
  for (int i = lane; i < full; i += 32) body[i] = make_uint4(0, 0, 0, 0);
  const int tail = head + full * V + lane;
  if (tail < dim) row[tail] = zero;
}
// beta times what is there
template <class O, int VE, class A>
__device__ inline void scale_row(O* row, int dim, A beta) {
  Sums<A, 8> zero;
  zero.clear();
  for (int c = 0; c < dim; c += kSelCols)
    store_axpby<O, VE, A, 8>(row, c, dim, zero, A(1), true, beta);
}

// A warp's queue of row parts on their way from global to shared memory.  Every lane copies and
// later reads its own pieces (of 16 bytes, or single elements of 4 or 8), so that no barrier is
// needed, and the bytes in flight do not cost registers.  Parts are asked for in batches: kStages
// batches of kBatch parts.  (With four or eight rows in flight in registers the combine reached
// half of the copy rate; it was waiting for latency with few warps, or short of registers.)
template <class P, int kBatch, int kStages> struct PartQueue {
  static constexpr int kPieces = P::U * P::N;
  static constexpr int kWarpBytes = kBatch * kStages * static_cast<int>(sizeof(P)) * 32;
  using Raw = typename P::Raw;
  Raw* base;      // this lane's first piece in stage 0; pieces of a lane are 32 apart
  int put, take;  // stages

  __device__ explicit PartQueue(unsigned char* warp_smem)
      : base(reinterpret_cast<Raw*>(warp_smem) + (threadIdx.x & 31)), put(0), take(0) {}
  __device__ static void copy(Raw* to, const void* from, bool live) {
    constexpr int kSize = static_cast<int>(sizeof(Raw));
    if constexpr (kSize == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to)), "l"(from),
                   "r"(live ? 16 : 0)
                   : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_addr(to)), "l"(from),
                   "n"(kSize), "r"(live ? kSize : 0)
                   : "memory");
  }
  // asks for part q of the batch being put together; a dead part becomes zeros
  template <class T> __device__ void push(int q, const T* row, bool live, int col0, int dim) {
    Raw* at = base + (put * kBatch + q) * (kPieces * 32);
#pragma unroll
    for (int u = 0; u < P::U; ++u) {
      const int c = P::column(col0, u);
#pragma unroll
      for (int p = 0; p < P::N; ++p)
        if (c < dim) copy(at + (u * P::N + p) * 32, row + c + p * P::OE, live);
    }
  }
  __device__ void send() {
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == kStages ? 0 : put + 1;
  }
  // waits for the oldest batch (kStages - 1 younger ones may still be under way)
  __device__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }
  __device__ P part(int q) const {
    const Raw* at = base + (take * kBatch + q) * (kPieces * 32);
    P v;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) v.r[i] = at[i * 32];
    return v;
  }
  __device__ void skip() { put = put + 1 == kStages ? 0 : put + 1; }  // shares another's groups
  // nothing may be under way when the warp ends
  __device__ void drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }
  __device__ void done() { take = take + 1 == kStages ? 0 : take + 1; }
};
// Four CTAs of eight warps share an SM, with 48 KB of queues each: 6 KB a warp, in batches of two
// parts of 1 KB (32 bytes a lane).
constexpr int kQueueCtas = 4;
constexpr int kQueueBatch = 2;
constexpr int kQueueStages = 3;
template <class T, int VE>
constexpr int kQueueCols = VE == 1 ? 8 : 32 / static_cast<int>(sizeof(T));  // of a lane
// whether parts can be queued: single 16-bit elements are too small for an asynchronous copy
template <class T, int VE> constexpr bool kQueued = VE * sizeof(T) >= 4;

// ---- embedding lookup ------------------------------------------------------------------------
// One warp per (token, group of G slabs): 2 KB of a 16-bit row in four loads a lane (16384 tokens,
// 131072 x 4096 bf16: 33 us, 5.8 TB/s; with two loads 36 us, with eight 33 us but odd widths 7.5
// instead of 5.1 us).  Lists too short for that many warps take one slab each (64 tokens: 2.0 us).
template <class T, class I, int VE, int G>
__global__ void __launch_bounds__(kSelThreads)
select_rows_kernel(IdKeys<I> ids, int64_t n, const T* table, int64_t ld_table,
                   int dim, T* out, int64_t ld_out,
                   typename acc_of<T>::type alpha, typename acc_of<T>::type beta, bool has_beta,
                   unsigned groups) {
  using A = typename acc_of<T>::type;
  follow();
  ids = behind(ids);
  table = behind(table);
  out = behind(out);
  const unsigned tb = blockIdx.x / groups, g = blockIdx.x - tb * groups;
  const int64_t i = static_cast<int64_t>(tb) * kSelWarps + (threadIdx.x >> 5);
  if (i >= n) return;
  const uint32_t id = ids(i);
  const bool live = id < ids.n_keys;
  const int col0 = static_cast<int>(g) * (G * kSelCols);
  Part<T, VE> r[G];
  if (live) {
#pragma unroll
    for (int s = 0; s < G; ++s)
      r[s].load(table + static_cast<int64_t>(id) * ld_table, col0 + s * kSelCols, dim);
  }
  T* o = out + i * ld_out;
#pragma unroll
  for (int s = 0; s < G; ++s) {
    Sums<A, 8> v;
    v.clear();
    if (live) v.set(r[s]);
    // (a masked row is zero whatever alpha is)
    store_axpby<T, VE, A, 8>(o, col0 + s * kSelCols, dim, v, live ? alpha : A(1), has_beta, beta);
  }
}

// ---- embedding gradient ----------------------------------------------------------------------
// The sorted (token, position) list is cut into ranges of some 24 entries (grad_ranges); a warp
// sums the rows of a range over one slab of columns and writes each token's row when its run of
// equal tokens ends.  A run that crosses a border and ends within 31 entries behind it is read to its
// end by the warp in front of the border.  A longer one is cut there: each range writes its piece
// as a partial row, and select_grad_long_kernel adds the pieces in order.  No floating-point
// atomics: the sums have one order whatever the scheduling.  Sums and pieces are float32 (float64)
// and rounded once, in the row of the result.
//
// What it measured: new gradient of 131072 x 2048 bf16 from 16384 tokens 104 us (5.8 TB/s, mostly
// zeros written; 14 us of it the sort); 32768 rows of 4096 bf16 added to 32000 x 4096 float32
// 131 us (4.3 TB/s: 14 us sort, 108 us sums, of whose issue slots 63 % are taken; two to six
// stages, and 16 or 32 bytes a lane, make no difference).  One range for every warp slot of the
// GPU took 150 us for these sums: a row that is read and written costs five times one that
// continues a run, so that equal numbers of entries are unequal work.
struct GradRuns {
  const Entry* list;  // tokens and their positions, sorted; the masked ones at the end
  int64_t n;
  uint32_t n_keys;
  __device__ uint32_t key(int64_t i) const { return list[i].key; }
};
// how many entries are not masked (made by whole warps)
__device__ inline int64_t grad_held(const GradRuns& runs) {
  if (runs.key(runs.n - 1) < runs.n_keys) return runs.n;
  int64_t lo = 0, len = runs.n;  // the answer is in [lo, lo + len)
  while (len > 0) {
    const int64_t step = (len + 31) / 32, end = lo + len;
    const int64_t at = lo + (threadIdx.x & 31) * step;
    const int hits = __popc(__ballot_sync(0xffffffffu, at < end && runs.key(at) < runs.n_keys));
    if (hits == 0) break;
    lo += (hits - 1) * step + 1;  // the entry in front of lo is held
    len = end - lo < step - 1 ? end - lo : step - 1;
  }
  return lo;
}
struct GradRange {
  int64_t range, size;  // its number, entries between two borders
  int64_t lo, hi;       // the entries it sums
  bool head, tail;      // its first run began before it; its last run goes on behind it
};

// The ranges of m entries: `most` of them, or fewer (of two entries at least).
struct GradRanges {
  int64_t m, size, count;
  __device__ GradRanges(int64_t held, int64_t most) : m(held) {
    const int64_t even = (held + most - 1) / most;
    size = even > 2 ? even : 2;
    count = (held + size - 1) / size;
  }
  __device__ int64_t border(int64_t r) const { return r * size < m ? r * size : m; }
};
// Entries from border x on that continue the run in front of it, kCross for that many or more.
// (With 64 fewer runs are cut, but the warp that reads on is late: 50257 x 771 float32 with a token
// on a third of 6001 places took 6 us more.)
constexpr int kCross = 32;
__device__ inline int grad_crossing(const GradRuns& runs, int64_t m, int64_t x) {
  if (x <= 0 || x >= m) return 0;
  const uint32_t key = runs.key(x - 1);
  int n = 0;
#pragma unroll
  for (int q = 0; q < kCross / 32; ++q) {
    const int64_t i = x + 32 * q + (threadIdx.x & 31);
    n += __popc(__ballot_sync(0xffffffffu, i < m && runs.key(i) == key));
  }
  return n;
}
__device__ inline GradRange grad_range(const GradRuns& runs, const GradRanges& all, int64_t r) {
  const int64_t a = all.border(r), b = all.border(r + 1);
  const int in = grad_crossing(runs, all.m, a), out = grad_crossing(runs, all.m, b);
  GradRange g;
  g.range = r;
  g.size = all.size;
  g.head = in == kCross;
  g.tail = out == kCross;
  g.lo = a + (g.head ? 0 : in);
  g.hi = b + (g.tail ? 0 : out);
  return g;
}

// Where the sums of a run go: its row of `out`, or a partial row of the range.
template <class T, class O> struct GradOut {
  using A = typename acc_of<T>::type;
  O* out;
  int64_t ld_out;
  A alpha, beta;
  A *head, *tail;  // partial rows of `dim` values, one per range
  int4* long_list;  // of each cut run: the ranges it begins and ends in, its token
  int32_t* long_count;
  int dim;

  // head: the run began before the range; tail: it goes on behind it
  template <int VE, int E, bool kBeta>
  __device__ void flush(const Sums<A, E>& acc, const Part<O, VE, E>& old, uint32_t key, int col0,
                        const GradRuns& runs, const GradRange& g, bool is_head,
                        bool is_tail) const {
    if (is_head)
      store_sums<A, VE>(head + g.range * dim, col0, dim, acc);
    else if (is_tail)
      store_sums<A, VE>(tail + g.range * dim, col0, dim, acc);
    else
      store_axpby<O, VE, A, E>(out + static_cast<int64_t>(key) * ld_out, col0, dim, acc, alpha,
                               kBeta, beta, old);
    if (is_head && !is_tail && col0 == 0) list(runs, g, key);
  }
  // a cut run ends in this range: where it begins (made by whole warps)
  __device__ void list(const GradRuns& runs, const GradRange& g, uint32_t key) const {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, len = g.lo;  // its first entry is in [lo, lo + len)
    while (len > 1) {
      const int64_t step = (len + 31) / 32, end = lo + len, at = lo + lane * step;
      const int below = __popc(__ballot_sync(0xffffffffu, at < end && runs.key(at) < key));
      if (below == 0) break;  // it is the entry at lo
      lo += (below - 1) * step + 1;
      len = end - lo < step ? end - lo : step;
    }
    // (the order of the list does not reach any result: every entry is finished by itself)
    if (lane == 0)
      long_list[atomicAdd(long_count, 1)] =
          make_int4(static_cast<int>(lo / g.size), static_cast<int>(g.range),
                    static_cast<int>(key), 0);
  }
};

// bit i: a run ends with entry i of the stretch whose keys the lanes hold
__device__ inline uint32_t run_ends(uint32_t keys, uint32_t next_keys) {
  const uint32_t first = __shfl_sync(0xffffffffu, next_keys, 0);
  uint32_t right = __shfl_down_sync(0xffffffffu, keys, 1);
  if ((threadIdx.x & 31) == 31) right = first;
  return __ballot_sync(0xffffffffu, right != keys);
}

// The rows of the range stream through the warp's queue; where `out` is added to, the row that a
// run ends in comes along with the run's last row (a run of one token, as most are, would
// otherwise wait for it by itself).  Keys and positions are read 32 at a time, a stretch ahead.
template <bool kBeta> constexpr int kGradStages = kBeta ? 4 : 6;
template <class T, class O, int VE, bool kBeta>
constexpr int kGradCols = kBeta && sizeof(O) > sizeof(T) ? 8 : kQueueCols<T, VE>;
template <class T, class O, int VE, bool kBeta>
__device__ inline void grad_sum(const GradRuns& runs, const GradRange& g,
                                const GradOut<T, O>& to, unsigned char* warp_smem, int col0,
                                const T* grad, int64_t ld_grad) {
  constexpr int E = kGradCols<T, O, VE, kBeta>, S = kGradStages<kBeta>;
  using Rows = PartQueue<Part<T, VE, E>, 1, S>;
  using Olds = PartQueue<Part<O, VE, E>, 1, S>;
  Rows rows(warp_smem);
  Olds olds(warp_smem + Rows::kWarpBytes);  // not touched unless kBeta
  const int lane = threadIdx.x & 31, dim = to.dim;
  const Entry* list = runs.list + g.lo;
  const int count = static_cast<int>(g.hi - g.lo);
  auto entry = [&](int i) { return i < count ? list[i] : Entry{0xffffffffu, 0}; };

  // the stretch that rows are asked for from and the one behind it; the keys of the stretch that
  // is summed and of the one behind it
  const Entry e0 = entry(lane), e1 = entry(32 + lane);
  int ask = 0, ask_pos = e0.pos, next_pos = e1.pos;
  uint32_t sum_keys = e0.key, next_keys = e1.key;
  uint32_t sum_ends = run_ends(sum_keys, next_keys);
  uint32_t ask_keys = sum_keys, ask_next = next_keys, ask_ends = sum_ends;
  bool ask_head = g.head, sum_head = g.head;
  auto send = [&] {
    const int at = ask & 31;
    const int64_t pos = __shfl_sync(0xffffffffu, ask_pos, at);
    if (ask < count) rows.push(0, grad + pos * ld_grad, true, col0, dim);
    if constexpr (kBeta) {
      const uint32_t key = __shfl_sync(0xffffffffu, ask_keys, at);
      if (ask < count && ((ask_ends >> at) & 1)) {
        if (!ask_head && !(g.tail && ask + 1 == count))
          olds.push(0, to.out + static_cast<int64_t>(key) * to.ld_out, true, col0, dim);
        ask_head = false;
      }
    }
    rows.send();
    if constexpr (kBeta) olds.skip();
    ++ask;
    if ((ask & 31) == 0) {
      const Entry e = entry(ask + 32 + lane);
      ask_pos = next_pos;
      next_pos = e.pos;
      if constexpr (kBeta) {
        ask_keys = ask_next;
        ask_next = e.key;
        ask_ends = run_ends(ask_keys, ask_next);
      }
    }
  };
  for (int q = 0; q < S - 1; ++q) send();
  Sums<typename acc_of<T>::type, E> acc;
  acc.clear();
  for (int i = 0; i < count; ++i) {
    send();
    rows.wait();
    acc.add(rows.part(0));
    const int at = i & 31;
    if ((sum_ends >> at) & 1) {
      Part<O, VE, E> old;
      if constexpr (kBeta) old = olds.part(0);
      to.template flush<VE, E, kBeta>(acc, old, __shfl_sync(0xffffffffu, sum_keys, at), col0,
                                      runs, g, sum_head, g.tail && i + 1 == count);
      acc.clear();
      sum_head = false;
    }
    rows.done();
    if constexpr (kBeta) olds.done();
    if (at == 31) {
      sum_keys = next_keys;
      next_keys = entry(i + 33 + lane).key;
      sum_ends = run_ends(sum_keys, next_keys);
    }
  }
  rows.drain();
}
// shared memory of one warp
template <class T, class O, int VE, bool kBeta>
constexpr int kGradWarpBytes =
    PartQueue<Part<T, VE, kGradCols<T, O, VE, kBeta>>, 1, kGradStages<kBeta>>::kWarpBytes +
    (kBeta ? PartQueue<Part<O, VE, kGradCols<T, O, VE, kBeta>>, 1, kGradStages<kBeta>>::kWarpBytes
           : 0);

// The same for 16-bit rows that cannot be taken 16 bytes at a time: groups of rows in registers.
template <class T, class O, bool kBeta>
__device__ inline void grad_sum_plain(const GradRuns& runs, const GradRange& g,
                                      const GradOut<T, O>& to, int col0,
                                      const T* grad, int64_t ld_grad) {
  constexpr int kAhead = 4;
  const int lane = threadIdx.x & 31;
  Sums<typename acc_of<T>::type, 8> acc;
  acc.clear();
  bool head = g.head;
  for (int64_t c = g.lo; c < g.hi; c += 32) {
    const Entry none{0xffffffffu, 0};
    const Entry e = c + lane < g.hi ? runs.list[c + lane] : none;
    const Entry f = c + 32 + lane < g.hi ? runs.list[c + 32 + lane] : none;
    const uint32_t keys = e.key, ends = run_ends(e.key, f.key);
    const int pos = e.pos;
    const int m = g.hi - c < 32 ? static_cast<int>(g.hi - c) : 32;
    for (int i0 = 0; i0 < m; i0 += kAhead) {
      Part<T, 1> r[kAhead];
      Part<O, 1> old[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int i = i0 + q;
        const int64_t p = __shfl_sync(0xffffffffu, pos, i & 31);
        const uint32_t key = __shfl_sync(0xffffffffu, keys, i & 31);
        if (i < m) {
          r[q].load(grad + p * ld_grad, col0, to.dim);
          if (kBeta && ((ends >> i) & 1))
            old[q].load(to.out + static_cast<int64_t>(key) * to.ld_out, col0, to.dim);
        }
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int i = i0 + q;
        const uint32_t key = __shfl_sync(0xffffffffu, keys, i & 31);
        if (i < m) {
          acc.add(r[q]);
          if ((ends >> i) & 1) {
            to.template flush<1, 8, kBeta>(acc, old[q], key, col0, runs, g, head,
                                           g.tail && c + i + 1 == g.hi);
            acc.clear();
            head = false;
          }
        }
      }
    }
  }
}

// CTAs that share an SM: as many as its 228 KB allow (a CTA takes 1 KB beside its queues), up to
// four; two where the rows are in registers.
constexpr int kSmemOfSm = 228 << 10;
template <class T, class O, int VE, bool kBeta>
constexpr int kGradCtas =
    !kQueued<T, VE>
        ? 2
        : std::min(kQueueCtas,
                   kSmemOfSm / (kSelWarps * kGradWarpBytes<T, O, VE, kBeta> + (1 << 10)));

// CTAs that sum and CTAs that write the rows no token names (zero, or beta times what is there;
// none when beta = 1 leaves them as they are) alternate from the first on, until one kind is used
// up: the waits of the first overlap the writes of the second, and no long CTA starts late.
// Rows per warp of the second kind.  Narrow accesses leave room for two CTAs on an SM, not four:
// their warps take four rows, whose flags are one load.
template <class T, int VE> constexpr int kRestRows = kQueued<T, VE> ? 1 : 4;
template <class T, class O, int VE, bool kBeta>
__global__ void __launch_bounds__(kSelThreads, kGradCtas<T, O, VE, kBeta>)
select_grad_kernel(GradRuns runs, int64_t ranges, unsigned sum_blocks, unsigned slabs,
                   const T* grad, int64_t ld_grad, GradOut<T, O> to,
                   const uint8_t* named) {
  extern __shared__ int4 smem4[];
  follow();
  runs.list = behind(runs.list);
  grad = behind(grad);
  to.out = behind(to.out);
  named = behind(named);
  const int warp = threadIdx.x >> 5;
  const unsigned b = blockIdx.x, rest = gridDim.x - sum_blocks;
  const unsigned both = 2 * (sum_blocks < rest ? sum_blocks : rest);
  const bool sums = b < both ? (b & 1) == 0 : sum_blocks > rest;
  const unsigned at = b < both ? b / 2 : b - both / 2;  // among the CTAs of its kind
  const int64_t w = static_cast<int64_t>(at) * kSelWarps + warp;
  if (!sums) {
    const int64_t row0 = w * kRestRows<T, VE>;
    if (row0 >= runs.n_keys) return;
    using Flags = typename raw_of<kRestRows<T, VE>>::type;
    const uint32_t flags = *reinterpret_cast<const Flags*>(named + row0);  // (padded)
    for (int q = 0; q < kRestRows<T, VE>; ++q) {
      if (((flags >> (8 * q)) & 1) || row0 + q >= runs.n_keys) continue;
      O* row = to.out + (row0 + q) * to.ld_out;
      if constexpr (kBeta) scale_row<O, VE>(row, to.dim, to.beta);
      else zero_row(row, to.dim);
    }
    return;
  }
  const int64_t range = w / slabs;
  const int slab = static_cast<int>(w - range * slabs);
  if (range >= ranges) return;
  const GradRanges all(grad_held(runs), ranges);
  if (range >= all.count) return;
  const GradRange g = grad_range(runs, all, range);
  if (g.lo >= g.hi) return;
  if constexpr (!kQueued<T, VE>)
    grad_sum_plain<T, O, kBeta>(runs, g, to, slab * kSelCols, grad, ld_grad);
  else
    grad_sum<T, O, VE, kBeta>(runs, g, to,
                              reinterpret_cast<unsigned char*>(smem4) +
                                  warp * kGradWarpBytes<T, O, VE, kBeta>,
                              slab * (32 * kGradCols<T, O, VE, kBeta>), grad, ld_grad);
}

// A run that was cut: the piece of the range it begins in, then the pieces of those behind.  One
// CTA per (run, slab of 32 E columns): its warps take the pieces in turn and the warps' sums are
// added in warp order.  The list names each run's first and last range, so that the sums wait for
// two loads in a row and no search (7 instead of 16 us for one run of 95 pieces).
constexpr int kLongWarps = 8;

template <class T, class O, int VE, int E>
__global__ void __launch_bounds__(32 * kLongWarps, sizeof(T) == 8 ? 2 : 3)
select_grad_long_kernel(GradOut<T, O> to, bool has_beta) {
  using A = typename acc_of<T>::type;
  __shared__ A sums[kLongWarps][E][32];
  follow();
  to.long_count = behind(to.long_count);
  to.long_list = behind(to.long_list);
  to.head = behind(to.head);
  to.tail = behind(to.tail);
  to.out = behind(to.out);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = *to.long_count;
  int4 run = to.long_list[blockIdx.x];  // (there is room for gridDim.x entries)
  const int col0 = static_cast<int>(blockIdx.y) * (32 * E);
  for (int item = blockIdx.x; item < count; item += gridDim.x) {
    if (item != static_cast<int>(blockIdx.x)) run = to.long_list[item];
    const int first = run.x, last = run.y;
    const uint32_t key = static_cast<uint32_t>(run.z);
    Sums<A, E> acc;
    acc.clear();
    constexpr int kAhead = 4;
    for (int r0 = first + warp; r0 <= last; r0 += kAhead * kLongWarps) {
      Part<A, VE, E> part[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const int r = r0 + q * kLongWarps;
        if (r <= last)
          part[q].load((r == first ? to.tail : to.head) + static_cast<int64_t>(r) * to.dim, col0,
                       to.dim);
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q)
        if (r0 + q * kLongWarps <= last) acc.add(part[q]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sums[warp][e][lane] = sum_of(acc, e);
    __syncthreads();
    if (warp == 0) {
      Sums<A, E> total;
      total.clear();
#pragma unroll
      for (int w = 0; w < kLongWarps; ++w) {
        Part<A, 1, E> part;
#pragma unroll
        for (int e = 0; e < E; ++e) part.set(e, sums[w][e][lane]);
        total.add(part);
      }
      store_axpby<O, VE, A, E>(to.out + static_cast<int64_t>(key) * to.ld_out, col0, to.dim, total,
                               to.alpha, has_beta, to.beta);
    }
    __syncthreads();
  }
}

// ---- tokens to experts and back ----------------------------------------------------------------
// a slot that names a row: masked ones are negative, and none may lead behind the array
__device__ inline bool is_row(int32_t s, int64_t rows) {
  return static_cast<uint32_t>(s) < static_cast<uint64_t>(rows);
}

// Rows are only moved: units of UB bytes, whatever the value type.  One warp per (token, slab);
// the token's row is read once and written to its slots.  The rows behind the last expert's are
// zeroed by the same warps.  (8192 tokens to 8 rows each, 4096 bf16: 94 us, 6.4 TB/s.)
template <int UB>
__global__ void __launch_bounds__(kSelThreads)
route_dispatch_kernel(const unsigned char* x, int64_t ld_x, int64_t n, int k,
                      int units, const int32_t* slots,
                      const int32_t* held_at, unsigned char* rows,
                      int64_t ld_rows, unsigned slabs) {
  using Raw = typename raw_of<UB>::type;
  constexpr int U = UB == 16 ? 4 : 8;
  follow();
  x = behind(x);
  slots = behind(slots);
  held_at = behind(held_at);
  const unsigned tb = blockIdx.x / slabs, slab = blockIdx.x - tb * slabs;
  const int64_t t = static_cast<int64_t>(tb) * kSelWarps + (threadIdx.x >> 5);
  if (t >= n) return;
  const int lane = threadIdx.x & 31, u0 = static_cast<int>(slab) * (32 * U) + lane;
  // the row, its slots and the number of rows held are asked for together
  Raw r[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u0 + 32 * u < units)
      r[u] = *reinterpret_cast<const Raw*>(x + t * ld_x + static_cast<int64_t>(u0 + 32 * u) * UB);
  int32_t my_slot = lane < k ? slots[t * k + lane] : -1;
  const int64_t held = *held_at;
  auto store = [&](int64_t row) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u0 + 32 * u < units)
        *reinterpret_cast<Raw*>(rows + row * ld_rows + (u0 + 32 * u) * int64_t{UB}) = r[u];
  };
  for (int j = 0; j < k; ++j) {
    if ((j & 31) == 0 && j > 0) my_slot = j + lane < k ? slots[t * k + j + lane] : -1;
    const int32_t s = __shfl_sync(0xffffffffu, my_slot, j & 31);
    if (is_row(s, n * k)) store(s);
  }
  memset(r, 0, sizeof(r));
  for (int64_t z = held + t; z < n * k; z += n) store(z);
}

// weights may be absent (1), of the value type, or float32
template <class T>
__device__ inline typename acc_of<T>::type route_weight(const void* w, bool w_is_f32, int64_t a) {
  using A = typename acc_of<T>::type;
  if (!w) return A(1);
  if (w_is_f32) return static_cast<A>(static_cast<const float*>(w)[a]);
  return to_acc(static_cast<const T*>(w)[a]);
}

// out[t] = alpha * sum_j w[t, j] * y[slots[t, j]] + beta * out[t].  A warp takes a range of tokens
// and one slab of columns; the assignments of its tokens are one stretch of `slots`, read 32 at a
// time and a stretch ahead, and their rows stream through the warp's queue without a pause
// between tokens.  A masked assignment is a part of zeros with weight zero; a token that has no
// other is beta * out whatever alpha is (alpha * 0 is not zero where alpha is not finite).
// (8192 x 8 rows of 4096 bf16: 101 us, 6.0 TB/s; 16384 x 4 rows of 2048: 55 us, 6.1 TB/s.  With 16
// bytes a lane and a wait for every row, 134 us: 82 % of the issue slots were taken.)
template <class T, int VE>
constexpr int kCombineCtas = VE == 1 && sizeof(T) == 8 ? 2 : kQueueCtas;
template <class T, int VE>
__global__ void __launch_bounds__(kSelThreads, kCombineCtas<T, VE>)
route_combine_kernel(const T* y, int64_t ld_y, const int32_t* slots,
                     const void* weights, bool w_is_f32, int64_t n, int k, int dim,
                     T* out, int64_t ld_out, typename acc_of<T>::type alpha,
                     typename acc_of<T>::type beta, bool has_beta, unsigned slabs,
                     unsigned ranges) {
  using A = typename acc_of<T>::type;
  constexpr int E = kQueueCols<T, VE>, B = kQueueBatch;
  using Queue = PartQueue<Part<T, VE, E>, B, kQueueStages>;
  extern __shared__ int4 smem4[];
  follow();
  y = behind(y);
  slots = behind(slots);
  weights = behind(weights);
  out = behind(out);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned w = blockIdx.x * kSelWarps + warp;
  const unsigned range = w / slabs, slab = w - range * slabs;
  if (range >= ranges) return;
  Queue queue(reinterpret_cast<unsigned char*>(smem4) + warp * Queue::kWarpBytes);
  const int col0 = static_cast<int>(slab) * (32 * E);
  int64_t t = n * range / ranges;
  const int64_t t1 = n * (range + 1) / ranges;
  const int32_t* my_slots = slots + t * k;
  const int64_t w0 = t * k;
  const int count = static_cast<int>((t1 - t) * k);  // the warp's assignments: 0 .. count - 1
  const uint32_t rows = static_cast<uint32_t>(n * k);

  // stretches of 32 assignments: the one that rows are asked for from, the one behind it; the
  // weights of the one that is summed from, and which of them are not masked, and of the one behind
  auto slot_of = [&](int a) {  // a valid slot, or -1
    const int32_t s = a < count ? my_slots[a] : -1;
    return static_cast<uint32_t>(s) < rows ? s : -1;
  };
  auto weight_of = [&](int a, uint32_t* live) {
    const bool held = slot_of(a) >= 0;
    *live = __ballot_sync(0xffffffffu, held);
    return held ? route_weight<T>(weights, w_is_f32, w0 + a) : A(0);
  };
  int32_t ask_slot = slot_of(lane), next_slot = slot_of(32 + lane);
  uint32_t live, next_live;
  A weight = weight_of(lane, &live), next_weight = weight_of(32 + lane, &next_live);
  int ask = 0;
  auto send = [&] {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      const int32_t s = __shfl_sync(0xffffffffu, ask_slot, (ask + q) & 31);
      if (y) queue.push(q, y + static_cast<int64_t>(s < 0 ? 0 : s) * ld_y, s >= 0, col0, dim);
    }
    queue.send();
    ask += B;
    if ((ask & 31) == 0) {
      ask_slot = next_slot;
      next_slot = slot_of(ask + 32 + lane);
    }
  };
  for (int q = 0; q < kQueueStages - 1; ++q) send();
  Sums<A, E> acc;
  acc.clear();
  if (k == 0)
    for (; t < t1; ++t)
      store_axpby<T, VE, A, E>(out + t * ld_out, col0, dim, acc, A(1), has_beta, beta);
  int j = 0;
  uint32_t any = 0;  // whether the token has an assignment that is not masked
  for (int a = 0; a < count; a += B) {
    send();
    if ((a & 31) == 0 && a > 0) {
      weight = next_weight;
      live = next_live;
      next_weight = weight_of(a + 32 + lane, &next_live);
    }
    queue.wait();
#pragma unroll
    for (int q = 0; q < B; ++q) {
      acc.fma(__shfl_sync(0xffffffffu, weight, (a + q) & 31), queue.part(q));
      any |= (live >> ((a + q) & 31)) & 1;
      if (++j == k) {
        if (a + q < count)
          store_axpby<T, VE, A, E>(out + t * ld_out, col0, dim, acc, any ? alpha : A(1), has_beta,
                                   beta);
        acc.clear();
        any = 0;
        j = 0;
        ++t;
      }
    }
    queue.done();
  }
  queue.drain();
}

// The same for 16-bit rows that cannot be taken 16 bytes at a time: one warp per (token, slab), up
// to 32 slots and weights read at once, four rows in flight in registers.
template <class T>
__global__ void __launch_bounds__(kSelThreads)
route_combine_plain_kernel(const T* y, int64_t ld_y,
                           const int32_t* slots, const void* weights,
                           bool w_is_f32, int64_t n, int k, int dim, T* out,
                           int64_t ld_out, typename acc_of<T>::type alpha,
                           typename acc_of<T>::type beta, bool has_beta, unsigned slabs) {
  using A = typename acc_of<T>::type;
  constexpr int kAhead = 4;
  follow();
  y = behind(y);
  slots = behind(slots);
  weights = behind(weights);
  out = behind(out);
  const unsigned tb = blockIdx.x / slabs, slab = blockIdx.x - tb * slabs;
  const int64_t t = static_cast<int64_t>(tb) * kSelWarps + (threadIdx.x >> 5);
  if (t >= n) return;
  const int lane = threadIdx.x & 31;
  const int col0 = static_cast<int>(slab) * kSelCols;
  Sums<A, 8> acc;
  acc.clear();
  bool any = false;  // whether the token has an assignment that is not masked
  for (int c = 0; c < k; c += 32) {
    int32_t my_slot = -1;
    A my_weight = A(0);
    if (c + lane < k) {
      my_slot = slots[t * k + c + lane];
      my_weight = route_weight<T>(weights, w_is_f32, t * k + c + lane);
    }
    const int m = k - c < 32 ? k - c : 32;
    for (int j0 = 0; j0 < m; j0 += kAhead) {
      Part<T, 1> r[kAhead];
      int32_t s[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        s[q] = __shfl_sync(0xffffffffu, my_slot, (j0 + q) & 31);
        if (j0 + q >= m) s[q] = -1;
        if (is_row(s[q], n * k)) r[q].load(y + static_cast<int64_t>(s[q]) * ld_y, col0, dim);
      }
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        const A w = __shfl_sync(0xffffffffu, my_weight, (j0 + q) & 31);
        if (is_row(s[q], n * k)) {
          acc.fma(w, r[q]);
          any = true;
        }
      }
    }
  }
  store_axpby<T, 1, A, 8>(out + t * ld_out, col0, dim, acc, any ? alpha : A(1), has_beta, beta);
}

// grad_y[slots[a]] = alpha * w[a] * g[a / k], grad_w[a] = alpha * <g[a / k], y[slots[a]]>: one
// warp per assignment a, over the whole row (the dot product ends in the warp); the warps of one
// token share its row of g through the caches.  Rows behind the last expert's are zeroed.  Held to
// 32 registers, so that 64 warps share an SM: 16384 x 4 rows of 2048 bf16 98 us, 6.2 TB/s (118 us
// with the 48 registers that the compiler takes otherwise).
template <class T, int VE>
__global__ void __launch_bounds__(kSelThreads, sizeof(T) < 8 ? 8 : 4)
route_combine_grad_kernel(const T* g, int64_t ld_g, const T* y,
                          int64_t ld_y, const int32_t* slots,
                          const int32_t* held_at,
                          const void* weights, bool w_is_f32, int64_t n, int k,
                          int dim, typename acc_of<T>::type alpha, T* grad_y,
                          int64_t ld_gy, void* grad_w) {
  using A = typename acc_of<T>::type;
  follow();
  g = behind(g);
  y = behind(y);
  slots = behind(slots);
  held_at = behind(held_at);
  weights = behind(weights);
  const int64_t a = blockIdx.x * static_cast<int64_t>(kSelWarps) + (threadIdx.x >> 5);
  if (a >= n * k) return;
  const int lane = threadIdx.x & 31;
  const int32_t s = slots[a];
  const int64_t z = *held_at + a;
  A dot = A(0);
  if (is_row(s, n * k)) {
    const T* gr = g + (a / k) * ld_g;
    const T* yr = y + static_cast<int64_t>(s) * ld_y;
    T* o = grad_y + static_cast<int64_t>(s) * ld_gy;
    const A w = alpha * route_weight<T>(weights, w_is_f32, a);
    for (int c = 0; c < dim; c += kSelCols) {
      Part<T, VE> rg, ry;
      rg.load(gr, c, dim);
      if (grad_w) ry.load(yr, c, dim);
      if (grad_w) {
#pragma unroll
        for (int u = 0; u < 8 / VE; ++u)
          if (Part<T, VE>::column(c, u) < dim) {
#pragma unroll
            for (int e = u * VE; e < u * VE + VE; ++e) fma_acc(dot, rg.get(e), ry.get(e));
          }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ry.set(e, w * rg.get(e));
      ry.store(o, c, dim);
    }
  }
  if (grad_w) {
    dot = group_sum(dot, 32);
    if (is_row(s, n * k)) dot = alpha * dot;  // (a masked one is zero whatever alpha is)
    if (lane == 0) {
      if (w_is_f32)
        static_cast<float*>(grad_w)[a] = static_cast<float>(dot);
      else
        static_cast<T*>(grad_w)[a] = storage_of<T>::from_acc(dot);
    }
  }
  if (z < n * k) zero_row(grad_y + z * ld_gy, dim);
}

// ---- host ----------------------------------------------------------------------------------------
#define B2S_DISPATCH_REAL(vtype, ...)                             \
  switch (vtype) {                                                \
    case B2S_F32: { using T = float; __VA_ARGS__; } break;        \
    case B2S_F64: { using T = double; __VA_ARGS__; } break;       \
    case B2S_F16: { using T = b2s::f16; __VA_ARGS__; } break;     \
    case B2S_BF16: { using T = b2s::bf16; __VA_ARGS__; } break;   \
    default: return B2S_ERR_DTYPE;                                \
  }

inline bool is_real(int vtype) {
  return vtype == B2S_F32 || vtype == B2S_F64 || vtype == B2S_F16 || vtype == B2S_BF16;
}
inline bool aligned_to(const void* p, size_t b) {
  return (reinterpret_cast<uintptr_t>(p) & (b - 1)) == 0;
}
// whether rows of `dim` values at p, ld values apart, can be taken 16 bytes at a time
inline bool wide_rows(const void* p, int64_t ld, int64_t dim, size_t es) {
  return aligned_to(p, 16) && (ld * es) % 16 == 0 && (dim * es) % 16 == 0;
}
// a row array: NULL only when it holds nothing; aligned to its elements; rows that do not overlap
inline int check_rows(const void* p, int64_t rows, int64_t ld, int64_t dim, size_t es) {
  if (rows <= 0 || dim <= 0) return B2S_OK;
  if (!p || (rows > 1 && ld < dim)) return B2S_ERR_ARG;
  return aligned_to(p, es) ? B2S_OK : B2S_ERR_ALIGNMENT;
}
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t kMaxGrid = 0x7fffffff;
#define B2S_TRY(expr)                    \
  do {                                   \
    const int st_ = (expr);              \
    if (st_ != B2S_OK) return st_;       \
  } while (0)

// How the sorted list is cut: ranges of 24 entries (rows that are also read and written take
// longer than others: the more ranges a warp slot gets, the more even the work; with ranges of 64
// the sums above took 127 us, with 16 the joining of runs grew by what they gained), longer ones
// where every slot has eight ranges already, and down to 2 entries where three quarters of the
// slots would have none (256 tokens: 7.7 us with ranges of 2, 10 us with 8).
inline int64_t grad_ranges(int64_t n, int64_t slabs, int64_t ctas_per_sm) {
  const int64_t slots = 148 * ctas_per_sm * kSelWarps;
  const int64_t most = std::min(8 * slots / slabs, ceil_div(n, 24));
  const int64_t least = std::min(slots / (4 * slabs), ceil_div(n, 2));
  return std::max<int64_t>(std::max(most, least), 1);
}
struct GradLayout {
  int64_t list, words, head, tail, named, end;
  int64_t ranges;  // partial rows there is room for
};
// words: the number of cut runs, the list of them
inline GradLayout grad_layout(int vtype, int64_t n, int64_t n_rows, int64_t dim) {
  GradLayout l;
  // (the most ranges any of the kernels uses: slabs of at most 1 KB, kQueueCtas CTAs)
  const int64_t slabs = ceil_div(dim * static_cast<int64_t>(vsize(vtype)), 1024);
  l.ranges = grad_ranges(n, slabs > 0 ? slabs : 1, kQueueCtas);
  const int64_t part = align256(l.ranges * dim * static_cast<int64_t>(acc_size(vtype)));
  int64_t at = sort_bytes(n, n_rows);
  l.list = at; at += align256(n * static_cast<int64_t>(sizeof(Entry)));
  l.words = at; at += align256((l.ranges + 1) * 16);
  l.head = at; at += part;
  l.tail = at; at += part;
  l.named = at; at += align256(n_rows);
  l.end = at;
  return l;
}

template <class T, class I>
int select_rows_run(const IdKeys<I>& ids, int64_t n, const void* table, int64_t ld_table,
                    int64_t dim, void* out, int64_t ld_out, double alpha, double beta,
                    cudaStream_t s) {
  using A = typename acc_of<T>::type;
  const bool wide = wide_rows(table, ld_table, dim, sizeof(T)) &&
                    wide_rows(out, ld_out, dim, sizeof(T));
  const int64_t slabs = ceil_div(dim, kSelCols), tbs = ceil_div(n, kSelWarps);
  const int G = tbs * slabs <= 148 * 8 ? 1 : 4;
  const int64_t groups = ceil_div(slabs, G), blocks = tbs * groups;
  if (blocks > kMaxGrid) return B2S_ERR_RANGE;
  const T* tp = static_cast<const T*>(table);
  T* op = static_cast<T*>(out);
  const A a = static_cast<A>(alpha), b = static_cast<A>(beta);
  auto go = [&](auto kernel) {
    return launch_behind(kernel, dim3(static_cast<unsigned>(blocks)), kSelThreads, 0, s, ids, n, tp,
                         ld_table, dim, op, ld_out, a, b, b != A(0), groups);
  };
  constexpr int VE = 16 / sizeof(T);
  if (wide)
    return G == 1 ? go(&select_rows_kernel<T, I, VE, 1>) : go(&select_rows_kernel<T, I, VE, 4>);
  return G == 1 ? go(&select_rows_kernel<T, I, 1, 1>) : go(&select_rows_kernel<T, I, 1, 4>);
}

template <class T, class O, int VE, bool kBeta>
int select_grad_go(const GradRuns& runs, const T* grad, int64_t ld_grad,
                   const GradOut<T, O>& to, const uint8_t* named, int64_t most_ranges,
                   cudaStream_t s) {
  using A = typename acc_of<T>::type;
  constexpr int E = kGradCols<T, O, VE, kBeta>;
  constexpr size_t smem = kQueued<T, VE> ? kSelWarps * kGradWarpBytes<T, O, VE, kBeta> : 0;
  constexpr int kCtas = kGradCtas<T, O, VE, kBeta>;
  static_assert(kCtas >= 1 && kCtas * (smem + (1 << 10)) <= kSmemOfSm);
  const int64_t slabs = ceil_div(to.dim, 32 * E);
  const int64_t ranges =
      runs.n == 0 ? 0
                  : std::min(grad_ranges(runs.n, slabs, kCtas), most_ranges);
  const int64_t sums = ceil_div(ranges * slabs, kSelWarps);
  const int64_t rest = to.beta == A(1) ? 0 : ceil_div(static_cast<int64_t>(runs.n_keys),
                                                        kRestRows<T, VE> * kSelWarps);
  if (sums + rest > kMaxGrid) return B2S_ERR_RANGE;
  if (sums + rest == 0) return B2S_OK;
  auto kernel = &select_grad_kernel<T, O, VE, kBeta>;
  if (smem > 0) ensure_dyn_smem(reinterpret_cast<const void*>(kernel), smem);
  B2S_TRY(launch_behind(kernel, dim3(static_cast<unsigned>(sums + rest)), kSelThreads, smem, s,
                        runs, ranges, sums, slabs, grad, ld_grad, to, named));
  if (runs.n > kCross) {  // a run that is cut goes on for kCross entries behind a border
    constexpr int kCols = VE > 1 && sizeof(T) == 8 ? 4 : 8;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(ranges, 128)),
                    static_cast<unsigned>(ceil_div(to.dim, 32 * kCols)));
    return launch_behind(&select_grad_long_kernel<T, O, VE, kCols>, grid, 32 * kLongWarps, 0, s, to,
                         kBeta);
  }
  return B2S_OK;
}

template <class T, class O>
int select_grad_run(const GradRuns& runs, const void* grad, int64_t ld_grad, int64_t dim, void* out,
                    int64_t ld_out, double alpha, double beta, unsigned char* ws,
                    const GradLayout& l, cudaStream_t s) {
  using A = typename acc_of<T>::type;
  const bool wide = wide_rows(grad, ld_grad, dim, sizeof(T)) &&
                    wide_rows(out, ld_out, dim, sizeof(O)) && (dim * sizeof(T)) % 16 == 0;
  int32_t* words = reinterpret_cast<int32_t*>(ws + l.words);
  const GradOut<T, O> to{static_cast<O*>(out), ld_out, static_cast<A>(alpha), static_cast<A>(beta),
                         reinterpret_cast<A*>(ws + l.head), reinterpret_cast<A*>(ws + l.tail),
                         reinterpret_cast<int4*>(words + 4), words, static_cast<int>(dim)};
  auto go = [&](auto run) {
    return run(runs, static_cast<const T*>(grad), ld_grad, to, ws + l.named, l.ranges, s);
  };
  constexpr int VE = 16 / sizeof(T);
  if (wide) return to.beta != A(0) ? go(&select_grad_go<T, O, VE, true>)
                                   : go(&select_grad_go<T, O, VE, false>);
  return to.beta != A(0) ? go(&select_grad_go<T, O, 1, true>) : go(&select_grad_go<T, O, 1, false>);
}

}  // namespace b2s

using namespace b2s;

extern "C" int b2s_select_rows(int val_type, int idx_type, const void* idx_dev, int64_t n,
                               int has_ignore, int64_t ignore, const void* table_dev,
                               int64_t n_rows, int64_t ld_table, int64_t dim, void* out_dev,
                               int64_t ld_out, double alpha, double beta, int32_t* status,
                               b2s_stream stream) {
  if (!is_real(val_type) || !isize(idx_type)) return B2S_ERR_DTYPE;
  if (n < 0 || n_rows < 0 || dim < 0) return B2S_ERR_ARG;
  if (n > kSortMaxEntries || n_rows > kSortMaxKeys || dim > kSelMaxDim) return B2S_ERR_RANGE;
  if (n == 0 || dim == 0) return B2S_OK;
  if (!idx_dev) return B2S_ERR_ARG;
  if (!aligned_to(idx_dev, isize(idx_type))) return B2S_ERR_ALIGNMENT;
  B2S_TRY(check_rows(table_dev, n_rows, ld_table, dim, vsize(val_type)));
  B2S_TRY(check_rows(out_dev, n, ld_out, dim, vsize(val_type)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  B2S_DISPATCH_I(idx_type, I, {
    const IdKeys<I> ids{static_cast<const I*>(idx_dev), static_cast<uint32_t>(n_rows),
                        has_ignore != 0, ignore, status};
    B2S_DISPATCH_REAL(val_type, return (select_rows_run<T, I>(ids, n, table_dev, ld_table, dim,
                                                              out_dev, ld_out, alpha, beta, s)));
  });
  return B2S_OK;
}

extern "C" int64_t b2s_select_grad_bytes(int val_type, int64_t n, int64_t n_rows, int64_t dim) {
  if (!is_real(val_type) || n < 0 || n_rows < 0 || dim < 0 || n > kSortMaxEntries ||
      n_rows > kSortMaxKeys || dim > kSelMaxDim)
    return 0;
  return grad_layout(val_type, n, n_rows, dim).end;
}

extern "C" int b2s_select_grad(int val_type, int out_type, int idx_type, const void* idx_dev,
                               int64_t n, int has_ignore, int64_t ignore, const void* grad_dev,
                               int64_t ld_grad, int64_t n_rows, int64_t dim, void* out_dev,
                               int64_t ld_out, double alpha, double beta, void* ws_dev,
                               int64_t ws_bytes, int32_t* status, b2s_stream stream) {
  if (!is_real(val_type) || !isize(idx_type)) return B2S_ERR_DTYPE;
  if (out_type != val_type && !(out_type == B2S_F32 && vsize(val_type) == 2)) return B2S_ERR_DTYPE;
  if (n < 0 || n_rows < 0 || dim < 0) return B2S_ERR_ARG;
  if (n > kSortMaxEntries || n_rows > kSortMaxKeys || dim > kSelMaxDim) return B2S_ERR_RANGE;
  if (n_rows == 0 || dim == 0) return B2S_OK;
  if (n > 0 && !idx_dev) return B2S_ERR_ARG;
  if (n > 0 && !aligned_to(idx_dev, isize(idx_type))) return B2S_ERR_ALIGNMENT;
  B2S_TRY(check_rows(grad_dev, n, ld_grad, dim, vsize(val_type)));
  B2S_TRY(check_rows(out_dev, n_rows, ld_out, dim, vsize(out_type)));
  const GradLayout l = grad_layout(val_type, n, n_rows, dim);
  if (!ws_dev || ws_bytes < l.end) return B2S_ERR_WORKSPACE;
  if (!aligned_to(ws_dev, 256)) return B2S_ERR_ALIGNMENT;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  unsigned char* ws = static_cast<unsigned char*>(ws_dev);
  Entry* list = reinterpret_cast<Entry*>(ws + l.list);
  int32_t* words = reinterpret_cast<int32_t*>(ws + l.words);
  B2S_DISPATCH_I(idx_type, I, {
    const IdKeys<I> ids{static_cast<const I*>(idx_dev), static_cast<uint32_t>(n_rows),
                        has_ignore != 0, ignore, status};
    const RunsOut sink{list, ws + l.named, static_cast<uint32_t>(n_rows)};
    B2S_TRY(sort_ids(ids, n, sink, ws + l.named, n_rows, words, ws, s));
  });
  const GradRuns runs{list, n, static_cast<uint32_t>(n_rows)};
  if (out_type == val_type) {
    B2S_DISPATCH_REAL(val_type, return (select_grad_run<T, T>(runs, grad_dev, ld_grad, dim,
                                                              out_dev, ld_out, alpha, beta, ws,
                                                              l, s)));
  } else if (val_type == B2S_F16) {
    return select_grad_run<f16, float>(runs, grad_dev, ld_grad, dim, out_dev, ld_out, alpha,
                                       beta, ws, l, s);
  } else {
    return select_grad_run<bf16, float>(runs, grad_dev, ld_grad, dim, out_dev, ld_out, alpha,
                                        beta, ws, l, s);
  }
  return B2S_OK;
}

extern "C" int64_t b2s_route_plan_bytes(int64_t n_tokens, int64_t k, int64_t n_experts) {
  if (n_tokens < 0 || k < 0 || n_experts < 0 || n_experts > kSortMaxBins - 1) return 0;
  if (k > 0 && n_tokens > kSortMaxEntries / k) return 0;
  return sort_bytes(n_tokens * k, n_experts);
}

extern "C" int b2s_route_plan(int idx_type, const void* experts_dev, int64_t n_tokens, int64_t k,
                              int64_t n_experts, int32_t* slots_dev, int32_t* indptr_dev,
                              int32_t* indices_dev, void* ws_dev, int64_t ws_bytes,
                              int32_t* status, b2s_stream stream) {
  if (!isize(idx_type)) return B2S_ERR_DTYPE;
  if (n_tokens < 0 || k < 0 || n_experts < 0 || !indptr_dev) return B2S_ERR_ARG;
  if (n_experts > kSortMaxBins - 1) return B2S_ERR_RANGE;
  if (k > 0 && n_tokens > kSortMaxEntries / k) return B2S_ERR_RANGE;
  const int64_t n = n_tokens * k;
  if (n > 0 && (!experts_dev || !slots_dev || !indices_dev)) return B2S_ERR_ARG;
  if (n > 0 && !aligned_to(experts_dev, isize(idx_type))) return B2S_ERR_ALIGNMENT;
  const int64_t need = sort_bytes(n, n_experts);
  if (ws_bytes < need || (need > 0 && !ws_dev)) return B2S_ERR_WORKSPACE;
  if (!aligned_to(ws_dev, 256)) return B2S_ERR_ALIGNMENT;
  B2S_DISPATCH_I(idx_type, I, {
    const IdKeys<I> ids{static_cast<const I*>(experts_dev), static_cast<uint32_t>(n_experts),
                        true, -1, status};
    const PlanOut sink{slots_dev, indptr_dev, indices_dev, static_cast<uint32_t>(n_experts),
                       static_cast<uint32_t>(k > 0 ? k : 1)};
    B2S_TRY(sort_ids(ids, n, sink, nullptr, 0, nullptr, static_cast<unsigned char*>(ws_dev),
                     static_cast<cudaStream_t>(stream)));
  });
  return B2S_OK;
}

namespace b2s {
inline int check_route(int val_type, int64_t n_tokens, int64_t k, int64_t dim,
                       const int32_t* slots) {
  if (!is_real(val_type)) return B2S_ERR_DTYPE;
  if (n_tokens < 0 || k < 0 || dim < 0) return B2S_ERR_ARG;
  if (dim > kSelMaxDim || (k > 0 && n_tokens > kSortMaxEntries / k)) return B2S_ERR_RANGE;
  if (n_tokens * k > 0 && !slots) return B2S_ERR_ARG;
  return B2S_OK;
}
inline int check_weights(int val_type, int w_type, const void* weights, bool* is_f32) {
  *is_f32 = false;
  if (!weights) return B2S_OK;
  if (w_type != val_type && w_type != B2S_F32) return B2S_ERR_DTYPE;
  if (!aligned_to(weights, vsize(w_type))) return B2S_ERR_ALIGNMENT;
  *is_f32 = w_type == B2S_F32;
  return B2S_OK;
}
template <class T, int VE>
int route_combine_go(const T* y, int64_t ld_y, const int32_t* slots, const void* weights,
                     bool w_f32, int64_t n, int64_t k, int64_t dim, T* out, int64_t ld_out,
                     double alpha, double beta, cudaStream_t s) {
  using A = typename acc_of<T>::type;
  auto kernel = &route_combine_kernel<T, VE>;
  constexpr int E = kQueueCols<T, VE>;
  constexpr size_t smem =
      kSelWarps * PartQueue<Part<T, VE, E>, kQueueBatch, kQueueStages>::kWarpBytes;
  ensure_dyn_smem(reinterpret_cast<const void*>(kernel), smem);
  const int64_t slabs = ceil_div(dim, 32 * E);
  // A range per warp that fits the GPU at once, and ranges of 16 rows where that makes more of
  // them: some SMs are a third faster than others at this, and take what the others leave (8192
  // x 8 rows of 4096 bf16: 101 us, 109 with one range a warp).
  constexpr int64_t kResident = 148 * kCombineCtas<T, VE> * kSelWarps;
  int64_t ranges = std::max<int64_t>(kResident / slabs, n * k / 16);
  ranges = ranges < 1 ? 1 : ranges > n ? n : ranges;
  // (a warp counts its assignments in 32 bits, a stretch or two behind the last: check_route has
  // held n * k to kSortMaxEntries, 2^25 below 2^31)
  const int64_t blocks = ceil_div(ranges * slabs, kSelWarps);
  if (blocks > kMaxGrid / kSelWarps) return B2S_ERR_RANGE;  // (warps are counted in 32 bits)
  const A b = static_cast<A>(beta);
  return launch_behind(kernel, dim3(static_cast<unsigned>(blocks)), kSelThreads, smem, s, y, ld_y,
                       slots, weights, w_f32, n, k, dim, out, ld_out, alpha, b, b != A(0), slabs,
                       ranges);
}

template <class T>
int route_combine_run(const void* y, int64_t ld_y, const int32_t* slots, const void* weights,
                      bool w_f32, int64_t n, int64_t k, int64_t dim, void* out, int64_t ld_out,
                      double alpha, double beta, cudaStream_t s) {
  const bool wide = wide_rows(out, ld_out, dim, sizeof(T)) &&
                    (k == 0 || wide_rows(y, ld_y, dim, sizeof(T)));
  const T* yp = static_cast<const T*>(y);
  T* op = static_cast<T*>(out);
  if (wide)
    return route_combine_go<T, 16 / sizeof(T)>(yp, ld_y, slots, weights, w_f32, n, k, dim, op,
                                               ld_out, alpha, beta, s);
  if constexpr (kQueued<T, 1>)
    return route_combine_go<T, 1>(yp, ld_y, slots, weights, w_f32, n, k, dim, op, ld_out, alpha,
                                  beta, s);
  if constexpr (!kQueued<T, 1>) {
    const int64_t slabs = ceil_div(dim, kSelCols), blocks = ceil_div(n, kSelWarps) * slabs;
    if (blocks > kMaxGrid) return B2S_ERR_RANGE;
    const float b = static_cast<float>(beta);
    return launch_behind(&route_combine_plain_kernel<T>, dim3(static_cast<unsigned>(blocks)),
                         kSelThreads, 0, s, yp, ld_y, slots, weights, w_f32, n, k, dim, op, ld_out,
                         alpha, b, b != 0, slabs);
  }
}

template <class T>
int route_combine_grad_run(const void* g, int64_t ld_g, const void* y, int64_t ld_y,
                           const int32_t* slots, const int32_t* held, const void* weights,
                           bool w_f32, int64_t n, int64_t k, int64_t dim, double alpha,
                           void* grad_y, int64_t ld_gy, void* grad_w, cudaStream_t s) {
  using A = typename acc_of<T>::type;
  const int64_t blocks = ceil_div(n * k, kSelWarps);
  if (blocks > kMaxGrid) return B2S_ERR_RANGE;
  const bool wide = wide_rows(g, ld_g, dim, sizeof(T)) &&
                    (!grad_w || wide_rows(y, ld_y, dim, sizeof(T))) &&
                    wide_rows(grad_y, ld_gy, dim, sizeof(T));
  auto go = [&](auto kernel) {
    return launch_behind(kernel, dim3(static_cast<unsigned>(blocks)), kSelThreads, 0, s,
                         static_cast<const T*>(g), ld_g, static_cast<const T*>(y), ld_y, slots,
                         held, weights, w_f32, n, k, dim, alpha, static_cast<T*>(grad_y), ld_gy,
                         grad_w);
  };
  return wide ? go(&route_combine_grad_kernel<T, 16 / sizeof(T)>)
              : go(&route_combine_grad_kernel<T, 1>);
}
}  // namespace b2s

extern "C" int b2s_route_dispatch(int val_type, const void* x_dev, int64_t ld_x, int64_t n_tokens,
                                  int64_t k, int64_t dim, const int32_t* slots_dev,
                                  const int32_t* held_dev, void* rows_dev, int64_t ld_rows,
                                  b2s_stream stream) {
  B2S_TRY(check_route(val_type, n_tokens, k, dim, slots_dev));
  const int64_t n = n_tokens * k;
  if (n == 0 || dim == 0) return B2S_OK;
  const size_t es = vsize(val_type);
  if (!held_dev) return B2S_ERR_ARG;
  B2S_TRY(check_rows(x_dev, n_tokens, ld_x, dim, es));
  B2S_TRY(check_rows(rows_dev, n, ld_rows, dim, es));
  const bool wide = wide_rows(x_dev, ld_x, dim, es) && wide_rows(rows_dev, ld_rows, dim, es);
  const int64_t units = wide ? dim * static_cast<int64_t>(es) / 16 : dim;
  const int64_t slabs = ceil_div(units, wide ? 128 : 256);
  const int64_t blocks = ceil_div(n_tokens, kSelWarps) * slabs;
  if (blocks > kMaxGrid) return B2S_ERR_RANGE;
  auto go = [&](auto kernel) {
    return launch_behind(kernel, dim3(static_cast<unsigned>(blocks)), kSelThreads, 0,
                         static_cast<cudaStream_t>(stream),
                         static_cast<const unsigned char*>(x_dev),
                         ld_x * static_cast<int64_t>(es), n_tokens, k, units, slots_dev, held_dev,
                         static_cast<unsigned char*>(rows_dev), ld_rows * static_cast<int64_t>(es),
                         slabs);
  };
  if (wide) return go(&route_dispatch_kernel<16>);
  return es == 2 ? go(&route_dispatch_kernel<2>)
                 : es == 4 ? go(&route_dispatch_kernel<4>) : go(&route_dispatch_kernel<8>);
}

extern "C" int b2s_route_combine(int val_type, const void* y_dev, int64_t ld_y,
                                 const int32_t* slots_dev, int w_type, const void* weights_dev,
                                 int64_t n_tokens, int64_t k, int64_t dim, void* out_dev,
                                 int64_t ld_out, double alpha, double beta, b2s_stream stream) {
  B2S_TRY(check_route(val_type, n_tokens, k, dim, slots_dev));
  if (n_tokens == 0 || dim == 0) return B2S_OK;
  bool w_f32;
  B2S_TRY(check_weights(val_type, w_type, weights_dev, &w_f32));
  B2S_TRY(check_rows(y_dev, n_tokens * k, ld_y, dim, vsize(val_type)));
  B2S_TRY(check_rows(out_dev, n_tokens, ld_out, dim, vsize(val_type)));
  B2S_DISPATCH_REAL(val_type, return (route_combine_run<T>(
      y_dev, ld_y, slots_dev, weights_dev, w_f32, n_tokens, k, dim, out_dev, ld_out, alpha, beta,
      static_cast<cudaStream_t>(stream))));
}

extern "C" int b2s_route_combine_grad(int val_type, const void* g_dev, int64_t ld_g,
                                      const void* y_dev, int64_t ld_y, const int32_t* slots_dev,
                                      const int32_t* held_dev, int w_type,
                                      const void* weights_dev, int64_t n_tokens, int64_t k,
                                      int64_t dim, double alpha, void* grad_y_dev, int64_t ld_gy,
                                      void* grad_w_dev, b2s_stream stream) {
  B2S_TRY(check_route(val_type, n_tokens, k, dim, slots_dev));
  const int64_t n = n_tokens * k;
  if (n == 0) return B2S_OK;
  if (!held_dev || (grad_w_dev && !weights_dev)) return B2S_ERR_ARG;
  bool w_f32;
  B2S_TRY(check_weights(val_type, w_type, weights_dev, &w_f32));
  B2S_TRY(check_weights(val_type, w_type, grad_w_dev, &w_f32));
  if (weights_dev) w_f32 = w_type == B2S_F32;
  B2S_TRY(check_rows(g_dev, n_tokens, ld_g, dim, vsize(val_type)));
  if (grad_w_dev) B2S_TRY(check_rows(y_dev, n, ld_y, dim, vsize(val_type)));
  B2S_TRY(check_rows(grad_y_dev, n, ld_gy, dim, vsize(val_type)));
  B2S_DISPATCH_REAL(val_type, return (route_combine_grad_run<T>(
      g_dev, ld_g, y_dev, ld_y, slots_dev, held_dev, weights_dev, w_f32, n_tokens, k, dim, alpha,
      grad_y_dev, ld_gy, grad_w_dev, static_cast<cudaStream_t>(stream))));
}
