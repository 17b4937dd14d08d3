// Products with a selection matrix that is never written out: the embedding lookup
// (Y = alpha S W + beta Y, S one-hot rows given by token ids), its gradient
// (dW = alpha S^T G + beta dW), and the routing of tokens to experts and back (S has k entries a
// row).  All of them move rows of `dim` values; a warp owns 256 columns of a row at a time, eight
// per lane, so that every load and store of a warp is one contiguous piece of a row.
#include "b2s_sort.cuh"

namespace b2s {

constexpr int kSelWarps = 8;            // warps per CTA of the row kernels
constexpr int kSelThreads = 32 * kSelWarps;
constexpr int kSelCols = 256;           // columns of a row a warp holds at a time (8 per lane)
constexpr int64_t kSelMaxDim = 1 << 22; // grids carry column slabs in their y / division

template <class T> struct acc_of { using type = float; };
template <> struct acc_of<double> { using type = double; };

template <int VB> struct raw_of;
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
// a row of zeros, or beta times what is there
template <class O, int VE, class A>
__device__ inline void scale_row(O* row, int dim, bool has_beta, A beta) {
  Sums<A, 8> zero;
  zero.clear();
  for (int c = 0; c < dim; c += kSelCols)
    store_axpby<O, VE, A, 8>(row, c, dim, zero, A(1), has_beta, beta);
}

// A warp's queue of row parts on their way from global to shared memory.  Every lane copies and
// later reads its own 16-byte pieces, so that no barrier is needed, and the bytes in flight do
// not cost registers.  Parts are asked for in batches: kStages batches of kBatch parts.
template <class P, int kBatch, int kStages> struct PartQueue {
  static constexpr int kPieces = P::U * P::N;
  static constexpr int kWarpBytes = kBatch * kStages * static_cast<int>(sizeof(P)) * 32;
  using Raw = typename P::Raw;
  Raw* base;      // this lane's first piece in stage 0; pieces of a lane are 32 apart
  int put, take;  // stages

  __device__ explicit PartQueue(unsigned char* warp_smem)
      : base(reinterpret_cast<Raw*>(warp_smem) + (threadIdx.x & 31)), put(0), take(0) {}
  // asks for part q of the batch being put together; a dead part becomes zeros
  template <class T> __device__ void push(int q, const T* row, bool live, int col0, int dim) {
    Raw* at = base + (put * kBatch + q) * (kPieces * 32);
#pragma unroll
    for (int u = 0; u < P::U; ++u) {
      const int c = P::column(col0, u);
#pragma unroll
      for (int p = 0; p < P::N; ++p)
        if (c < dim)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                           smem_addr(at + (u * P::N + p) * 32)),
                       "l"(row + c + p * P::OE), "r"(live ? 16 : 0)
                       : "memory");
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
  // nothing may be under way when the warp ends
  __device__ void drain() { asm volatile("cp.async.wait_all;" ::: "memory"); }
  __device__ void done() { take = take + 1 == kStages ? 0 : take + 1; }
};
// Four CTAs of eight warps share an SM, with 48 KB of queues each: 6 KB a warp, in batches of two
// parts of 1 KB (32 bytes a lane).
constexpr int kQueueCtas = 4;
constexpr int kQueueBatch = 2;
constexpr int kQueueStages = 3;
template <class T> constexpr int kQueueCols = 32 / static_cast<int>(sizeof(T));  // of a lane

// ---- embedding lookup ------------------------------------------------------------------------
// One warp per (token, group of G slabs).
template <class T, class I, int VE, int G>
__global__ void __launch_bounds__(kSelThreads)
select_rows_kernel(IdKeys<I> ids, int64_t n, const T* __restrict__ table, int64_t ld_table,
                   int dim, T* __restrict__ out, int64_t ld_out,
                   typename acc_of<T>::type alpha, typename acc_of<T>::type beta, bool has_beta,
                   unsigned groups) {
  using A = typename acc_of<T>::type;
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
    if (live) v.add(r[s]);
    // (a masked row is zero whatever alpha is)
    store_axpby<T, VE, A, 8>(o, col0 + s * kSelCols, dim, v, live ? alpha : A(1), has_beta, beta);
  }
}

// ---- embedding gradient ----------------------------------------------------------------------
// The sorted (token, position) list is cut into tiles of 32 entries; a warp sums the rows of one
// tile over one slab of columns and writes each token's row when its run of equal tokens ends.
// A run that begins in one tile and ends in the next belongs to the first (it reads on); only a
// run that spans two borders or more is written as one partial row per tile, which
// select_grad_long_kernel adds in tile order.  No floating-point atomics: the sums have one
// order whatever the scheduling.
constexpr int kGradTile = 32;

struct GradRuns {
  const uint32_t* keys;  // sorted tokens; n_keys: masked, at the end
  const int32_t* vals;   // their positions
  int64_t n;
  uint32_t n_keys;
};

__device__ inline uint32_t run_key(const GradRuns& g, int64_t i) {
  return (i >= 0 && i < g.n) ? g.keys[i] : (i < 0 ? 0xffffffffu : g.n_keys);
}

template <class T, class O, int VE>
__device__ inline void grad_tile(const GradRuns& runs, int64_t tile, int slab,
                                 const T* __restrict__ grad, int64_t ld_grad, int dim,
                                 O* __restrict__ out, int64_t ld_out,
                                 typename acc_of<T>::type alpha, typename acc_of<T>::type beta,
                                 bool has_beta, typename acc_of<T>::type* __restrict__ head,
                                 typename acc_of<T>::type* __restrict__ tail,
                                 int32_t* __restrict__ long_list, int32_t* long_count) {
  using A = typename acc_of<T>::type;
  using RP = Part<T, VE>;
  constexpr int P = kGradTile;
  const int lane = threadIdx.x & 31;
  const int64_t at = tile * P;
  const uint32_t none = runs.n_keys;
  const uint32_t cur = run_key(runs, at + lane);
  const uint32_t nxt = run_key(runs, at + P + lane);
  const uint32_t prv = run_key(runs, at - P + lane);
  const int valid = __popc(__ballot_sync(0xffffffffu, cur < none));
  if (valid == 0) return;
  const uint32_t before = __shfl_sync(0xffffffffu, prv, 31);  // key of the entry before the tile
  const uint32_t last = __shfl_sync(0xffffffffu, cur, valid - 1);
  const uint32_t after = __shfl_sync(0xffffffffu, nxt, 0);
  const int in_head = __popc(__ballot_sync(0xffffffffu, cur == before));
  const int in_prev = __popc(__ballot_sync(0xffffffffu, prv == before));
  const int in_tail = __popc(__ballot_sync(0xffffffffu, cur == last));
  const int in_next = __popc(__ballot_sync(0xffffffffu, nxt == last));
  const bool head_ends = in_head < P || after != before;
  const bool head_began = in_prev < P || run_key(runs, at - P - 1) != before;
  const bool goes_on = valid == P && after == last;
  const bool tail_begins = in_tail < P || before != last;
  const bool tail_ends = in_next < P || run_key(runs, at + 2 * P) != last;
  const bool own_head = in_head > 0 && !(head_ends && head_began);  // a piece of a long run
  const int lo = (in_head > 0 && !own_head) ? in_head : 0;
  const bool long_tail = goes_on && tail_begins && !tail_ends;
  const int hi = valid + (goes_on && tail_begins && tail_ends ? in_next : 0);
  if (lo >= hi) return;
  if (long_tail && slab == 0 && lane == 0) {
    // (the order of the list does not reach any result: every entry is finished by itself)
    long_list[atomicAdd(long_count, 1)] = static_cast<int32_t>(tile);
  }
  const int pos_cur = at + lane < runs.n ? runs.vals[at + lane] : 0;
  const int pos_nxt = at + P + lane < runs.n ? runs.vals[at + P + lane] : 0;
  const int col0 = slab * kSelCols;

  Sums<A, 8> acc;
  acc.clear();
  // The rows of a group, and the rows of `out` that its ends are added to, are all asked for
  // before the first is used: a run of one token (most are) would otherwise wait for its old
  // row by itself.
  constexpr int kAhead = 4;
  for (int i0 = lo; i0 < hi; i0 += kAhead) {
    RP r[kAhead];
    Part<O, VE> old[kAhead];
    uint32_t key[kAhead];
    bool ends[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int i = i0 + q;
      const int a = __shfl_sync(0xffffffffu, pos_cur, i & 31);
      const int b = __shfl_sync(0xffffffffu, pos_nxt, i & 31);
      const uint32_t ka = __shfl_sync(0xffffffffu, cur, i & 31);
      const uint32_t kb = __shfl_sync(0xffffffffu, cur, (i + 1) & 31);
      key[q] = i < P ? ka : last;
      ends[q] = i < hi && (i + 1 >= hi || (i + 1 < P ? kb : last) != key[q]);
      if (i < hi) r[q].load(grad + static_cast<int64_t>(i < P ? a : b) * ld_grad, col0, dim);
      const bool part = (own_head && i < in_head) || (long_tail && i + 1 == hi);
      if (has_beta && ends[q] && !part)
        old[q].load(out + static_cast<int64_t>(key[q]) * ld_out, col0, dim);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int i = i0 + q;
      if (i < hi) {
        acc.add(r[q]);
        if (ends[q]) {
          const bool is_head = own_head && i < in_head;
          if (is_head || (long_tail && i + 1 == hi)) {
            A* part = (is_head ? head : tail) + tile * dim;
            store_sums<A, VE>(part, col0, dim, acc);
          } else {
            store_axpby<O, VE, A, 8>(out + static_cast<int64_t>(key[q]) * ld_out, col0, dim, acc,
                                     alpha, has_beta, beta, old[q]);
          }
          acc.clear();
        }
      }
    }
  }
}

// CTAs that sum tiles and CTAs that write the rows no token names (zero, or beta times what is
// there; none when beta = 1 leaves them as they are) alternate from the first on, until one kind
// is used up: the waits of the first overlap the writes of the second, and no long CTA starts
// late.
template <class T, class O, int VE>
__global__ void __launch_bounds__(kSelThreads)
select_grad_kernel(GradRuns runs, int64_t n_tiles, unsigned sum_blocks, unsigned slabs,
                   const T* __restrict__ grad, int64_t ld_grad, int dim, O* __restrict__ out,
                   int64_t ld_out, typename acc_of<T>::type alpha, typename acc_of<T>::type beta,
                   bool has_beta, typename acc_of<T>::type* __restrict__ head,
                   typename acc_of<T>::type* __restrict__ tail, int32_t* __restrict__ long_list,
                   int32_t* long_count, const uint8_t* __restrict__ named) {
  const int warp = threadIdx.x >> 5;
  const unsigned b = blockIdx.x, rest = gridDim.x - sum_blocks;
  const unsigned both = 2 * (sum_blocks < rest ? sum_blocks : rest);
  const bool sums = b < both ? (b & 1) == 0 : sum_blocks > rest;
  const unsigned at = b < both ? b / 2 : b - both / 2;  // among the CTAs of its kind
  if (sums) {
    const unsigned tb = at / slabs, slab = at - tb * slabs;
    const int64_t tile = static_cast<int64_t>(tb) * kSelWarps + warp;
    if (tile < n_tiles)
      grad_tile<T, O, VE>(runs, tile, static_cast<int>(slab), grad, ld_grad, dim, out, ld_out,
                          alpha, beta, has_beta, head, tail, long_list, long_count);
    return;
  }
  const int64_t row = static_cast<int64_t>(at) * kSelWarps + warp;
  if (row < runs.n_keys && !named[row]) scale_row<O, VE>(out + row * ld_out, dim, has_beta, beta);
}

// A run that spans two tile borders or more: the piece of its first tile, then the pieces of the
// tiles behind it.  One CTA per (run, 128 columns): its warps take the pieces in turn and the
// warps' sums are added in warp order.
constexpr int kLongWarps = 8;
constexpr int kLongCols = 128;

template <class A, class O>
__global__ void __launch_bounds__(32 * kLongWarps)
select_grad_long_kernel(GradRuns runs, int64_t n_tiles, int dim, O* __restrict__ out,
                        int64_t ld_out, A alpha, A beta, bool has_beta,
                        const A* __restrict__ head, const A* __restrict__ tail,
                        const int32_t* __restrict__ long_list,
                        const int32_t* __restrict__ long_count) {
  __shared__ A sums[kLongWarps][kLongCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = *long_count;
  const int col0 = static_cast<int>(blockIdx.y) * kLongCols + lane;
  for (int item = blockIdx.x; item < count; item += gridDim.x) {
    const int64_t first = long_list[item];
    const uint32_t key = runs.keys[first * kGradTile + kGradTile - 1];
    // the last tile whose first entry has this key, 32 places at a time
    int64_t lo = first + 1, len = n_tiles - lo;
    while (len > 1) {
      const int64_t step = (len + 31) / 32;
      const int64_t at = lo + lane * step;
      const bool mine = at < lo + len && runs.keys[at * kGradTile] <= key;
      const int hits = __popc(__ballot_sync(0xffffffffu, mine));  // lane 0 always hits
      const int64_t end = lo + len;
      lo += (hits - 1) * step;
      len = end - lo < step ? end - lo : step;
    }
    A acc[4] = {A(0), A(0), A(0), A(0)};
#pragma unroll 4
    for (int64_t t = first + warp; t <= lo; t += kLongWarps) {
      const A* part = (t == first ? tail : head) + t * dim;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col0 + 32 * e < dim) acc[e] = acc[e] + part[col0 + 32 * e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    if (threadIdx.x < kLongCols) {
      A s = A(0);
#pragma unroll
      for (int w = 0; w < kLongWarps; ++w) s = s + sums[w][threadIdx.x];
      const int col = static_cast<int>(blockIdx.y) * kLongCols + threadIdx.x;
      if (col < dim) {
        O* o = out + static_cast<int64_t>(key) * ld_out + col;
        A x = alpha * s;
        if (has_beta) x = x + beta * static_cast<A>(to_acc(*o));
        *o = storage_of<O>::from_acc(x);
      }
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
// zeroed by the same warps.
template <int UB>
__global__ void __launch_bounds__(kSelThreads)
route_dispatch_kernel(const unsigned char* __restrict__ x, int64_t ld_x, int64_t n, int k,
                      int units, const int32_t* __restrict__ slots,
                      const int32_t* __restrict__ held_at, unsigned char* __restrict__ rows,
                      int64_t ld_rows, unsigned slabs) {
  using Raw = typename raw_of<UB>::type;
  constexpr int U = UB == 16 ? 4 : 8;
  const unsigned tb = blockIdx.x / slabs, slab = blockIdx.x - tb * slabs;
  const int64_t t = static_cast<int64_t>(tb) * kSelWarps + (threadIdx.x >> 5);
  if (t >= n) return;
  const int u0 = static_cast<int>(slab) * (32 * U) + (threadIdx.x & 31);
  Raw r[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u0 + 32 * u < units)
      r[u] = *reinterpret_cast<const Raw*>(x + t * ld_x + static_cast<int64_t>(u0 + 32 * u) * UB);
  for (int j = 0; j < k; ++j) {
    const int32_t s = slots[t * k + j];
    if (!is_row(s, n * k)) continue;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u0 + 32 * u < units)
        *reinterpret_cast<Raw*>(rows + s * ld_rows + static_cast<int64_t>(u0 + 32 * u) * UB) = r[u];
  }
  memset(r, 0, sizeof(r));
  for (int64_t z = *held_at + t; z < n * k; z += n) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u0 + 32 * u < units)
        *reinterpret_cast<Raw*>(rows + z * ld_rows + static_cast<int64_t>(u0 + 32 * u) * UB) = r[u];
  }
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
// between tokens.  A masked assignment is a part of zeros with weight zero.
template <class T, int VE>
__global__ void __launch_bounds__(kSelThreads, kQueueCtas)
route_combine_kernel(const T* __restrict__ y, int64_t ld_y, const int32_t* __restrict__ slots,
                     const void* __restrict__ weights, bool w_is_f32, int64_t n, int k, int dim,
                     T* __restrict__ out, int64_t ld_out, typename acc_of<T>::type alpha,
                     typename acc_of<T>::type beta, bool has_beta, unsigned slabs,
                     unsigned ranges) {
  using A = typename acc_of<T>::type;
  constexpr int E = kQueueCols<T>, B = kQueueBatch;
  using Queue = PartQueue<Part<T, VE, E>, B, kQueueStages>;
  extern __shared__ int4 smem4[];
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
  // weights of the one that is summed from, and of the one behind it
  auto slot_of = [&](int a) {  // a valid slot, or -1
    const int32_t s = a < count ? my_slots[a] : -1;
    return static_cast<uint32_t>(s) < rows ? s : -1;
  };
  auto weight_of = [&](int a) {
    return slot_of(a) >= 0 ? route_weight<T>(weights, w_is_f32, w0 + a) : A(0);
  };
  int32_t ask_slot = slot_of(lane), next_slot = slot_of(32 + lane);
  A weight = weight_of(lane), next_weight = weight_of(32 + lane);
  int ask = 0;
  auto send = [&] {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      const int32_t s = __shfl_sync(0xffffffffu, ask_slot, (ask + q) & 31);
      queue.push(q, y + static_cast<int64_t>(s < 0 ? 0 : s) * ld_y, s >= 0, col0, dim);
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
  int j = 0;
  for (int a = 0; a < count; a += B) {
    send();
    if ((a & 31) == 0 && a > 0) {
      weight = next_weight;
      next_weight = weight_of(a + 32 + lane);
    }
    queue.wait();
#pragma unroll
    for (int q = 0; q < B; ++q) {
      acc.fma(__shfl_sync(0xffffffffu, weight, (a + q) & 31), queue.part(q));
      if (++j == k) {
        if (a + q < count)
          store_axpby<T, VE, A, E>(out + t * ld_out, col0, dim, acc, alpha, has_beta, beta);
        acc.clear();
        j = 0;
        ++t;
      }
    }
    queue.done();
  }
  queue.drain();
}

// The same for rows that cannot be taken 16 bytes at a time: one warp per (token, slab), up to 32
// slots and weights read at once, four rows in flight in registers.
template <class T>
__global__ void __launch_bounds__(kSelThreads)
route_combine_plain_kernel(const T* __restrict__ y, int64_t ld_y,
                           const int32_t* __restrict__ slots, const void* __restrict__ weights,
                           bool w_is_f32, int64_t n, int k, int dim, T* __restrict__ out,
                           int64_t ld_out, typename acc_of<T>::type alpha,
                           typename acc_of<T>::type beta, bool has_beta, unsigned slabs) {
  using A = typename acc_of<T>::type;
  constexpr int kAhead = 4;
  const unsigned tb = blockIdx.x / slabs, slab = blockIdx.x - tb * slabs;
  const int64_t t = static_cast<int64_t>(tb) * kSelWarps + (threadIdx.x >> 5);
  if (t >= n) return;
  const int lane = threadIdx.x & 31;
  const int col0 = static_cast<int>(slab) * kSelCols;
  Sums<A, 8> acc;
  acc.clear();
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
        if (is_row(s[q], n * k)) acc.fma(w, r[q]);
      }
    }
  }
  store_axpby<T, 1, A, 8>(out + t * ld_out, col0, dim, acc, alpha, has_beta, beta);
}

// grad_y[slots[a]] = alpha * w[a] * g[a / k], grad_w[a] = alpha * <g[a / k], y[slots[a]]>: one
// warp per assignment a, over the whole row (the dot product ends in the warp); the warps of one
// token share its row of g through the caches.  Rows behind the last expert's are zeroed.
template <class T, int VE>
__global__ void __launch_bounds__(kSelThreads, sizeof(T) < 8 ? 8 : 4)
route_combine_grad_kernel(const T* __restrict__ g, int64_t ld_g, const T* __restrict__ y,
                          int64_t ld_y, const int32_t* __restrict__ slots,
                          const int32_t* __restrict__ held_at,
                          const void* __restrict__ weights, bool w_is_f32, int64_t n, int k,
                          int dim, typename acc_of<T>::type alpha, T* __restrict__ grad_y,
                          int64_t ld_gy, void* __restrict__ grad_w) {
  using A = typename acc_of<T>::type;
  const int64_t a = blockIdx.x * static_cast<int64_t>(kSelWarps) + (threadIdx.x >> 5);
  if (a >= n * k) return;
  const int lane = threadIdx.x & 31;
  const int32_t s = slots[a];
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
    dot = alpha * group_sum(dot, 32);
    if (lane == 0) {
      if (w_is_f32)
        static_cast<float*>(grad_w)[a] = static_cast<float>(dot);
      else
        static_cast<T*>(grad_w)[a] = storage_of<T>::from_acc(dot);
    }
  }
  const int64_t z = *held_at + a;
  if (z < n * k) scale_row<T, VE, A>(grad_y + z * ld_gy, dim, false, A(0));
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

struct GradLayout {
  int64_t keys, vals, list, head, tail, named, end;
};
inline GradLayout grad_layout(int vtype, int64_t n, int64_t n_rows, int64_t dim) {
  GradLayout l;
  const int64_t tiles = ceil_div(n, kGradTile);
  int64_t at = sort_bytes(n, n_rows);
  l.keys = at; at += align256(n * 4);
  l.vals = at; at += align256(n * 4);
  l.list = at; at += align256((tiles + 1) * 4);
  l.head = at; at += align256(tiles * dim * static_cast<int64_t>(acc_size(vtype)));
  l.tail = at; at += align256(tiles * dim * static_cast<int64_t>(acc_size(vtype)));
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
#define B2S_GO(VE, GG)                                                                          \
  select_rows_kernel<T, I, VE, GG><<<static_cast<unsigned>(blocks), kSelThreads, 0, s>>>(       \
      ids, n, tp, ld_table, static_cast<int>(dim), op, ld_out, a, b, b != A(0),                 \
      static_cast<unsigned>(groups))
  if (wide) {
    if (G == 1) B2S_GO(16 / sizeof(T), 1); else B2S_GO(16 / sizeof(T), 4);
  } else {
    if (G == 1) B2S_GO(1, 1); else B2S_GO(1, 4);
  }
#undef B2S_GO
  return launch_status();
}

template <class T, class O>
int select_grad_run(const GradRuns& runs, const void* grad, int64_t ld_grad, int64_t dim,
                    void* out, int64_t ld_out, double alpha, double beta, unsigned char* ws,
                    const GradLayout& l, cudaStream_t s) {
  using A = typename acc_of<T>::type;
  const bool wide = wide_rows(grad, ld_grad, dim, sizeof(T)) &&
                    wide_rows(out, ld_out, dim, sizeof(O)) && (dim * sizeof(T)) % 16 == 0;
  const int64_t tiles = ceil_div(runs.n, kGradTile), slabs = ceil_div(dim, kSelCols);
  const A a = static_cast<A>(alpha), b = static_cast<A>(beta);
  const int64_t sums = ceil_div(tiles, kSelWarps) * slabs;
  const int64_t rest = b == A(1) ? 0 : ceil_div(static_cast<int64_t>(runs.n_keys), kSelWarps);
  if (sums + rest > kMaxGrid) return B2S_ERR_RANGE;
  if (sums + rest == 0) return B2S_OK;
  A* head = reinterpret_cast<A*>(ws + l.head);
  A* tail = reinterpret_cast<A*>(ws + l.tail);
  int32_t* list = reinterpret_cast<int32_t*>(ws + l.list);
  const unsigned grid = static_cast<unsigned>(sums + rest);
#define B2S_GO(VE)                                                                             \
  select_grad_kernel<T, O, VE><<<grid, kSelThreads, 0, s>>>(                                   \
      runs, tiles, static_cast<unsigned>(sums), static_cast<unsigned>(slabs),                  \
      static_cast<const T*>(grad), ld_grad, static_cast<int>(dim), static_cast<O*>(out), ld_out, \
      a, b, b != A(0), head, tail, list + 1, list, ws + l.named)
  if (wide) B2S_GO(16 / sizeof(T)); else B2S_GO(1);
#undef B2S_GO
  if (tiles > 2) {  // a long run touches three tiles at least
    const dim3 lg(static_cast<unsigned>(tiles < 256 ? tiles : 256),
                  static_cast<unsigned>(ceil_div(dim, kLongCols)));
    select_grad_long_kernel<A, O><<<lg, 32 * kLongWarps, 0, s>>>(
        runs, tiles, static_cast<int>(dim), static_cast<O*>(out), ld_out, a, b, b != A(0), head,
        tail, list + 1, list);
  }
  return launch_status();
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
  uint32_t* keys = reinterpret_cast<uint32_t*>(ws + l.keys);
  int32_t* vals = reinterpret_cast<int32_t*>(ws + l.vals);
  B2S_DISPATCH_I(idx_type, I, {
    const IdKeys<I> ids{static_cast<const I*>(idx_dev), static_cast<uint32_t>(n_rows),
                        has_ignore != 0, ignore, status};
    const RunsOut sink{keys, vals, ws + l.named, static_cast<uint32_t>(n_rows)};
    B2S_TRY(sort_ids(ids, n, sink, ws + l.named, n_rows,
                     reinterpret_cast<int32_t*>(ws + l.list), ws, s));
  });
  const GradRuns runs{keys, vals, n, static_cast<uint32_t>(n_rows)};
  if (out_type == val_type) {
    B2S_DISPATCH_REAL(val_type, return (select_grad_run<T, T>(runs, grad_dev, ld_grad, dim,
                                                              out_dev, ld_out, alpha, beta, ws,
                                                              l, s)));
  } else if (val_type == B2S_F16) {
    return select_grad_run<f16, float>(runs, grad_dev, ld_grad, dim, out_dev, ld_out, alpha, beta,
                                       ws, l, s);
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
  if (!ws_dev || ws_bytes < sort_bytes(n, n_experts)) return B2S_ERR_WORKSPACE;
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
  constexpr int E = kQueueCols<T>;
  constexpr size_t smem =
      kSelWarps * PartQueue<Part<T, VE, E>, kQueueBatch, kQueueStages>::kWarpBytes;
  ensure_dyn_smem(reinterpret_cast<const void*>(kernel), smem);
  const int64_t slabs = ceil_div(dim, 32 * E);
  // every warp that fits the GPU at once gets one range
  constexpr int64_t kResident = 148 * kQueueCtas * kSelWarps;
  int64_t ranges = kResident / slabs;
  ranges = ranges < 1 ? 1 : ranges > n ? n : ranges;
  // a warp counts its assignments in 32 bits (with two stretches to spare)
  while (ceil_div(n, ranges) * k > 0x7fff0000) ++ranges;
  const int64_t blocks = ceil_div(ranges * slabs, kSelWarps);
  const A b = static_cast<A>(beta);
  kernel<<<static_cast<unsigned>(blocks), kSelThreads, smem, s>>>(
      y, ld_y, slots, weights, w_f32, n, static_cast<int>(k), static_cast<int>(dim), out, ld_out,
      static_cast<A>(alpha), b, b != A(0), static_cast<unsigned>(slabs),
      static_cast<unsigned>(ranges));
  return launch_status();
}

template <class T>
int route_combine_run(const void* y, int64_t ld_y, const int32_t* slots, const void* weights,
                      bool w_f32, int64_t n, int64_t k, int64_t dim, void* out, int64_t ld_out,
                      double alpha, double beta, cudaStream_t s) {
  const bool wide = k > 0 && wide_rows(y, ld_y, dim, sizeof(T)) &&
                    wide_rows(out, ld_out, dim, sizeof(T));
  const T* yp = static_cast<const T*>(y);
  T* op = static_cast<T*>(out);
  if (wide)
    return route_combine_go<T, 16 / sizeof(T)>(
        yp, ld_y, slots, weights, w_f32, n, k, dim, op, ld_out, alpha, beta, s);
  using A = typename acc_of<T>::type;
  const int64_t slabs = ceil_div(dim, kSelCols), blocks = ceil_div(n, kSelWarps) * slabs;
  if (blocks > kMaxGrid) return B2S_ERR_RANGE;
  const A b = static_cast<A>(beta);
  route_combine_plain_kernel<T><<<static_cast<unsigned>(blocks), kSelThreads, 0, s>>>(
      yp, ld_y, slots, weights, w_f32, n, static_cast<int>(k), static_cast<int>(dim), op, ld_out,
      static_cast<A>(alpha), b, b != A(0), static_cast<unsigned>(slabs));
  return launch_status();
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
    kernel<<<static_cast<unsigned>(blocks), kSelThreads, 0, s>>>(
        static_cast<const T*>(g), ld_g, static_cast<const T*>(y), ld_y, slots, held, weights,
        w_f32, n, static_cast<int>(k), static_cast<int>(dim), static_cast<A>(alpha),
        static_cast<T*>(grad_y), ld_gy, grad_w);
    return launch_status();
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
#define B2S_GO(VB)                                                                             \
  route_dispatch_kernel<VB><<<static_cast<unsigned>(blocks), kSelThreads, 0,                   \
                              static_cast<cudaStream_t>(stream)>>>(                            \
      static_cast<const unsigned char*>(x_dev), ld_x * static_cast<int64_t>(es), n_tokens,     \
      static_cast<int>(k), static_cast<int>(units), slots_dev, held_dev,                       \
      static_cast<unsigned char*>(rows_dev), ld_rows * static_cast<int64_t>(es),               \
      static_cast<unsigned>(slabs))
  if (wide) B2S_GO(16);
  else if (es == 2) B2S_GO(2);
  else if (es == 4) B2S_GO(4);
  else B2S_GO(8);
#undef B2S_GO
  return launch_status();
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
