// Stable counting sort of ids: tokens by vocabulary row (embedding gradient), assignments by
// expert (token route).  Least significant digit first; one digit of up to 11 bits per pass, so
// that a route needs one pass and a vocabulary of 2^17 rows two.
//
// A list of up to 8192 entries is sorted in one launch by a cluster of eight CTAs (up to 1024: by
// one CTA), which read each other's digit counts through distributed shared memory (6001 entries
// in two passes: 10 us).  Where an SM has more entries, its scattered stores are the limit: 16384
// took 64 us on one SM, 17 us on eight, and 14 us in three launches.  The passes of a longer list
// cut it into at most 128 chunks, one CTA each.
// The first kernel counts the digits of each chunk; the second sums those counts itself (every CTA
// reads the whole chunks x digits table, which L2 holds), places its entries in order and counts
// the next digit of each in the chunk that it is placed in.
#pragma once
#include <type_traits>

#include "b2s_tile.cuh"

namespace b2s {

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortRounds = 1;                           // entries per thread and tile
constexpr int kSortTile = kSortThreads * kSortRounds;
constexpr int kSortMaxChunks = 128;
constexpr int kTeamThreads = 1024;                       // CTAs of a cluster that sorts alone
constexpr int kTeamWarps = kTeamThreads / 32;
constexpr int kTeamCtas = 8;
constexpr int64_t kTeamMost = kTeamThreads * kTeamCtas;
constexpr int kSortMaxBits = 11;
constexpr int kSortMaxBins = 1 << kSortMaxBits;
constexpr int64_t kSortMaxEntries = 0x7fffffff - (1 << 25);  // positions are int32
constexpr int64_t kSortMaxKeys = 0x7ffffffe;             // n_keys itself stands for masked

inline int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

// Caller's ids -> keys: 0 .. n_keys - 1, or n_keys for a masked id (sorted behind all others).
// An id outside the range that is not the masked one is treated as masked and reported.
template <class I> struct IdKeys {
  const I* ids;
  uint32_t n_keys;
  bool has_ignore;
  int64_t ignore;
  int32_t* status;  // may be NULL; host-visible word, set (not ORed) on error

  __device__ uint32_t operator()(int64_t i) const {
    const int64_t id = static_cast<int64_t>(ids[i]);
    if (has_ignore && id == ignore) return n_keys;
    if (static_cast<uint64_t>(id) >= n_keys) {
      if (status) *reinterpret_cast<volatile int32_t*>(status) = 1 << B2S_ERR_BOUNDS;
      return n_keys;
    }
    return static_cast<uint32_t>(id);
  }
};

// A sorted entry: its key and its position in the caller's list.  The two are stored together: the
// scattered stores are what a pass waits for.
struct __align__(8) Entry {
  uint32_t key;
  int32_t pos;
};
__device__ inline Entry load_entry(const Entry* p) {
  const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p));
  return {v.x, static_cast<int32_t>(v.y)};
}

// Where a pass takes its entries from: the caller's ids, or the list of the pass before.
template <class I> struct FromIds {
  IdKeys<I> key;
  __device__ Entry operator()(int64_t i) const { return {key(i), static_cast<int32_t>(i)}; }
};
struct FromList {
  const Entry* list;
  __device__ Entry operator()(int64_t i) const { return load_entry(list + i); }
};

// ---- where the sorted entries go ---------------------------------------------------------------
struct ListOut {  // between two passes
  Entry* list;
  __device__ void operator()(Entry e, int dst) const { list[dst] = e; }
  __device__ void first(int, int) const {}
};
struct RunsOut {  // embedding gradient: the sorted list, and which rows are named at all
  static constexpr bool kOnePass = false;
  Entry* list;
  uint8_t* named;
  uint32_t n_keys;
  __device__ void operator()(Entry e, int dst) const {
    list[dst] = e;
    if (e.key < n_keys) named[e.key] = 1;
  }
  __device__ void first(int, int) const {}
};
struct PlanOut {  // token route: slot of each assignment, token of each slot, first slot per expert
  static constexpr bool kOnePass = true;  // its keys fit one digit: no kernel for a second pass,
                                          // and first() needs the counts of a digit
  int32_t* slots;
  int32_t* indptr;
  int32_t* indices;
  uint32_t n_experts, k;
  __device__ void operator()(Entry e, int dst) const {
    slots[e.pos] = e.key < n_experts ? dst : -1;
    indices[dst] = static_cast<int32_t>(static_cast<uint32_t>(e.pos) / k);
  }
  __device__ void first(int bin, int at) const {
    if (bin <= static_cast<int>(n_experts)) indptr[bin] = at;
  }
};

// ---- kernels that follow each other --------------------------------------------------------------
// Each kernel is put in place while the one before it in the stream still runs (programmatic
// dependent launch), which hides its launch: 1 to 2 us of each.  Every thread of every kernel calls
// follow() before it touches memory or ends: it returns when the kernel before has ended and its
// writes are visible, and lets the kernel behind be put in place.
__device__ inline void follow() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
// A pointer as it is known behind follow().  What is read through it cannot be read before (the
// compiler may move loads that it takes for constant in front of a wait; a pointer that it knows
// nothing of until then leaves it nothing to move).
template <class T> __device__ inline T* behind(T* p) {
  asm volatile("" : "+l"(p)::"memory");
  return p;
}
template <class I> __device__ inline IdKeys<I> behind(IdKeys<I> ids) {
  ids.ids = behind(ids.ids);
  return ids;
}
template <class I> __device__ inline FromIds<I> behind(FromIds<I> from) {
  from.key = behind(from.key);
  return from;
}
__device__ inline FromList behind(FromList from) {
  from.list = behind(from.list);
  return from;
}
// launches `kernel`, which calls follow()
template <class... Params, class... Args>
int launch_behind(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                  const Args&... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = smem;
  config.stream = st;
  config.attrs = &early;
  config.numAttrs = 1;
  cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
  return launch_status();  // (reads and clears the error of a launch that was refused)
}

// ---- device pieces of a pass ---------------------------------------------------------------------
// counts the digits of entries [lo, hi) into hist[bins] (shared, zeroed by the caller)
template <class From>
__device__ inline void sort_count(const From& from, int64_t lo, int64_t hi, int shift, int bins,
                                  int* hist) {
  const int lane = threadIdx.x & 31;
  for (int64_t i0 = lo; i0 < hi; i0 += kSortThreads) {
    const int64_t i = i0 + threadIdx.x;
    unsigned d = 0xffffffffu;
    if (i < hi) d = (from(i).key >> shift) & (bins - 1);
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    if (i < hi && (peers & ((1u << lane) - 1u)) == 0) atomicAdd(hist + d, __popc(peers));
  }
}

// exclusive prefix sum of v[bins] (shared) in place, by kThreads threads; bins <= kSortMaxBins
template <int kThreads>
__device__ inline void sort_scan(int* v, int bins, int* warp_tot) {
  constexpr int kPer = kSortMaxBins / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int c[kPer], run = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int b = threadIdx.x * kPer + q;
    c[q] = b < bins ? v[b] : 0;
    run += c[q];
  }
  int inc = run;
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) warp_tot[warp] = inc;
  __syncthreads();
  int in_front = lane < warp ? warp_tot[lane] : 0;
  for (int o = 16; o > 0; o >>= 1) in_front += __shfl_xor_sync(0xffffffffu, in_front, o);
  int at = in_front + inc - run;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int b = threadIdx.x * kPer + q;
    if (b < bins) v[b] = at;
    at += c[q];
  }
  __syncthreads();
}

// Rank of the lane's entry among those of the warp so far that have the same digit (0xffffffff:
// no entry); `mine` counts them.
__device__ inline int sort_rank(unsigned digit, uint16_t* mine) {
  const unsigned peers = __match_any_sync(0xffffffffu, digit);
  const int before = __popc(peers & ((1u << (threadIdx.x & 31)) - 1u));
  const bool live = digit != 0xffffffffu;
  int prev = 0;
  if (live) prev = mine[digit];
  __syncwarp();
  if (live && before == 0) mine[digit] = static_cast<uint16_t>(prev + __popc(peers));
  __syncwarp();
  return prev + before;
}

// The counts of the pass behind: entry by entry, where it is placed (integer sums: any order).
struct NextCounts {
  int* table;  // NULL: there is no pass behind
  unsigned chunk;
  int shift;
  __device__ void operator()(const Entry& e, int dst, int bins) const {
    if (table)
      atomicAdd(table + static_cast<int64_t>(dst / chunk) * bins + ((e.key >> shift) & (bins - 1)),
                1);
  }
};

// Places entries [lo, hi) in order; off[b] is where the next entry with digit b goes.  A warp
// takes 32 neighbouring entries per round: those with the same digit are ranked by lane, the
// rounds and warps of a tile by the counters cnt[warp][digit], tiles by off.
template <class From, class Out>
__device__ inline void sort_place(const From& from, const Out& out, int64_t lo, int64_t hi,
                                  int shift, int bins, int* off, int* off_next, uint16_t* cnt,
                                  const NextCounts& next) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t t0 = lo; t0 < hi; t0 += kSortTile) {
    uint32_t* z = reinterpret_cast<uint32_t*>(cnt);
    for (int i = threadIdx.x; i < kSortWarps * bins / 2; i += kSortThreads) z[i] = 0;
    __syncthreads();
    Entry e[kSortRounds];
    int rank[kSortRounds];
    uint16_t* mine = cnt + warp * bins;
#pragma unroll
    for (int q = 0; q < kSortRounds; ++q) {
      const int64_t i = t0 + (warp * kSortRounds + q) * 32 + lane;
      const bool live = i < hi;
      if (live) e[q] = from(i);
      rank[q] = sort_rank(live ? (e[q].key >> shift) & (bins - 1) : 0xffffffffu, mine);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {
      int run = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = cnt[w * bins + b];
        cnt[w * bins + b] = static_cast<uint16_t>(run);
        run += c;
      }
      off_next[b] = off[b] + run;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kSortRounds; ++q) {
      const int64_t i = t0 + (warp * kSortRounds + q) * 32 + lane;
      if (i < hi) {
        const int d = (e[q].key >> shift) & (bins - 1);
        const int dst = off[d] + mine[d] + rank[q];
        out(e[q], dst);
        next(e[q], dst, bins);
      }
    }
    int* swap = off;
    off = off_next;
    off_next = swap;
    __syncthreads();
  }
}

// shared memory of a pass: off, off_next (int[bins] each), cnt (uint16[warps][bins])
inline size_t sort_smem(int bins) {
  return static_cast<size_t>(bins) * (2 * sizeof(int) + kSortWarps * sizeof(uint16_t));
}

// ---- kernels -------------------------------------------------------------------------------------
// counts[chunk][digit] of the first digit; the CTAs also zero the tables of the others behind it,
// `clear` (flags of the caller) and *counter
template <class I>
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(FromIds<I> from, int64_t n, int64_t chunk, int bins, int passes, int* counts,
                  uint8_t* clear, int64_t n_clear, int32_t* counter) {
  extern __shared__ int4 smem4[];
  int* hist = reinterpret_cast<int*>(smem4);
  follow();
  from = behind(from);
  for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
  __syncthreads();
  const int64_t lo = blockIdx.x * chunk, hi = lo + chunk < n ? lo + chunk : n;
  sort_count(from, lo, hi, 0, bins, hist);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kSortThreads;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kSortThreads) + threadIdx.x;
       i < (n_clear + 15) / 16; i += stride)
    reinterpret_cast<uint4*>(clear)[i] = make_uint4(0, 0, 0, 0);
  if (counter && blockIdx.x == 0 && threadIdx.x == 0) *counter = 0;
  const int64_t table = static_cast<int64_t>(gridDim.x) * bins;
  for (int64_t i = table + blockIdx.x * static_cast<int64_t>(kSortThreads) + threadIdx.x;
       i < passes * table; i += stride)
    counts[i] = 0;
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kSortThreads)
    counts[blockIdx.x * static_cast<int64_t>(bins) + b] = hist[b];
}

template <class From, class Out>
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(From from, Out out, int64_t n, int64_t chunk, int shift, int bins,
                  const int* counts, NextCounts next) {
  extern __shared__ int4 smem4[];
  __shared__ int warp_tot[kSortWarps];
  follow();
  from = behind(from);
  counts = behind(counts);
  int* off = reinterpret_cast<int*>(smem4);
  int* before = off + bins;  // off_next until the first tile
  uint16_t* cnt = reinterpret_cast<uint16_t*>(before + bins);
  for (int b = threadIdx.x; b < bins; b += kSortThreads) off[b] = before[b] = 0;
  __syncthreads();
  // every group of bins / 4 threads sums some of the chunks (integer sums: any order)
  const int quads = bins / 4, groups = kSortThreads / quads > 0 ? kSortThreads / quads : 1;
  const int group = threadIdx.x / quads, quad = threadIdx.x - group * quads;
  if (group < groups) {
    int4 all = make_int4(0, 0, 0, 0), pre = make_int4(0, 0, 0, 0);
    const int4* table = reinterpret_cast<const int4*>(counts);
    const int chunks = gridDim.x, me = blockIdx.x;
#pragma unroll 8
    for (int c = group; c < chunks; c += groups) {
      const int4 v = table[static_cast<int64_t>(c) * quads + quad];
      all.x += v.x; all.y += v.y; all.z += v.z; all.w += v.w;
      if (c < me) { pre.x += v.x; pre.y += v.y; pre.z += v.z; pre.w += v.w; }
    }
    atomicAdd(off + 4 * quad, all.x); atomicAdd(off + 4 * quad + 1, all.y);
    atomicAdd(off + 4 * quad + 2, all.z); atomicAdd(off + 4 * quad + 3, all.w);
    atomicAdd(before + 4 * quad, pre.x); atomicAdd(before + 4 * quad + 1, pre.y);
    atomicAdd(before + 4 * quad + 2, pre.z); atomicAdd(before + 4 * quad + 3, pre.w);
  }
  __syncthreads();
  sort_scan<kSortThreads>(off, bins, warp_tot);
  for (int b = threadIdx.x; b < bins; b += kSortThreads) {
    if (blockIdx.x == 0) out.first(b, off[b]);
    off[b] += before[b];
  }
  __syncthreads();
  const int64_t lo = blockIdx.x * chunk, hi = lo + chunk < n ? lo + chunk : n;
  sort_place(from, out, lo, hi, shift, bins, off, before, cnt, next);
}

// All CTAs of the cluster, and their memory accesses before it
__device__ inline void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// *p of the CTA `rank` of the cluster (p: shared memory here, the same place there)
__device__ inline int cluster_load(const int* p, unsigned rank) {
  uint32_t at;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// A list that a cluster sorts (gridDim.x CTAs, all of one cluster).  CTA c takes `chunk` entries, a
// thread one of them, so that (CTA, warp, lane) is the order of the list.  The counters of the
// warps are summed per digit in place, those of the CTAs through distributed shared memory.
template <class I, class Out>
__global__ void __launch_bounds__(kTeamThreads)
sort_team_kernel(FromIds<I> ids, Out out, int n, int chunk, int bits, int passes, Entry* list0,
                 Entry* list1, uint8_t* clear, int64_t n_clear, int32_t* counter) {
  extern __shared__ int4 smem4[];
  __shared__ int warp_tot[kTeamWarps];
  follow();
  ids = behind(ids);
  const int bins = 1 << bits, warp = threadIdx.x >> 5;
  const unsigned me = blockIdx.x, ctas = gridDim.x;
  int* off = reinterpret_cast<int*>(smem4);
  int* total = off + bins;                                     // of this CTA, read by the others
  uint32_t* cnt2 = reinterpret_cast<uint32_t*>(total + bins);  // two 16-bit counters a word
  uint16_t* mine = reinterpret_cast<uint16_t*>(cnt2) + warp * bins;
  const int lo = static_cast<int>(me) * chunk, hi = n - lo < chunk ? n : lo + chunk;
  const int i = lo + static_cast<int>(threadIdx.x);  // this thread's entry
  for (int64_t c = me * kTeamThreads + threadIdx.x; c < (n_clear + 15) / 16;
       c += ctas * kTeamThreads)
    reinterpret_cast<uint4*>(clear)[c] = make_uint4(0, 0, 0, 0);
  if (counter && me == 0 && threadIdx.x == 0) *counter = 0;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    Entry e{0, 0};
    if (i < hi) {
      if (Out::kOnePass || p == 0) e = ids(i);
      else e = load_entry(((p & 1) ? list0 : list1) + i);  // what pass p - 1 wrote
    }
    const unsigned digit = (e.key >> shift) & (bins - 1);
    for (int c = threadIdx.x; c < kTeamWarps * bins / 2; c += kTeamThreads) cnt2[c] = 0;
    __syncthreads();
    const int rank = sort_rank(i < hi ? digit : 0xffffffffu, mine);
    __syncthreads();
    for (int b = threadIdx.x; b < bins / 2; b += kTeamThreads) {
      uint32_t run = 0;
#pragma unroll 8
      for (int w = 0; w < kTeamWarps; ++w) {
        const uint32_t c = cnt2[w * (bins / 2) + b];
        cnt2[w * (bins / 2) + b] = run;
        run += c;
      }
      total[2 * b] = run & 0xffff;
      total[2 * b + 1] = run >> 16;
    }
    cluster_barrier();
    int before[kSortMaxBins / kTeamThreads];
#pragma unroll
    for (int u = 0; u < kSortMaxBins / kTeamThreads; ++u) {
      const int b = threadIdx.x + u * kTeamThreads;
      before[u] = 0;
      if (b < bins) {
        int all = 0;
        for (unsigned c = 0; c < ctas; ++c) {
          const int v = cluster_load(total + b, c);
          all += v;
          if (c < me) before[u] += v;
        }
        off[b] = all;
      }
    }
    __syncthreads();
    sort_scan<kTeamThreads>(off, bins, warp_tot);
    const bool last = p + 1 == passes;
#pragma unroll
    for (int u = 0; u < kSortMaxBins / kTeamThreads; ++u) {
      const int b = threadIdx.x + u * kTeamThreads;
      if (b < bins) {
        if (last && me == 0) out.first(b, off[b]);
        off[b] += before[u];
      }
    }
    __syncthreads();
    if (i < hi) {
      const int dst = rank + off[digit] + mine[digit];
      if (Out::kOnePass || last) out(e, dst);
      else ((p & 1) ? list1 : list0)[dst] = e;
    }
    // what was placed is read by other CTAs, and no CTA may end or count anew while its counts are
    cluster_barrier();
  }
}

// A list of at most kFewMost entries: every thread counts the entries that stand before its own,
// in a time that grows with their square.  Whole gradients of 512 bf16 columns added to float32, by
// counting and by the cluster kernel: 2000 rows (one digit) 64 entries 6.4 and 9.8 us, 256 15.6 and
// 17.0, 320 17.7 and 17.5, 512 22.6 and 17.9; 32000 rows (two digits) 64 entries 5.9 and 10.3 us,
// 256 12.0 and 14.5, 384 16.2 and 16.6, 512 21.9 and 18.7, 1024 49.4 and 22.6.
constexpr int kFewMost = 256;
template <class I, class Out>
__global__ void __launch_bounds__(kFewMost)
sort_few_kernel(FromIds<I> ids, Out out, int n, uint8_t* clear, int64_t n_clear,
                int32_t* counter) {
  __shared__ __align__(16) uint32_t keys[kFewMost];
  follow();
  ids = behind(ids);
  const int i = threadIdx.x;
  const Entry mine = i < n ? ids(i) : Entry{0xffffffffu, 0};
  keys[i] = mine.key;
  for (int64_t c = i; c < (n_clear + 15) / 16; c += kFewMost)
    reinterpret_cast<uint4*>(clear)[c] = make_uint4(0, 0, 0, 0);
  if (counter && i == 0) *counter = 0;
  __syncthreads();
  if (i >= n) return;
  int before = 0;
  for (int j = 0; j < n; j += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(keys + j);  // (behind n: the largest)
    before += k.x < mine.key || (k.x == mine.key && j < i);
    before += k.y < mine.key || (k.y == mine.key && j + 1 < i);
    before += k.z < mine.key || (k.z == mine.key && j + 2 < i);
    before += k.w < mine.key || (k.w == mine.key && j + 3 < i);
  }
  out(mine, before);
}

// flags that are too many for the cluster
__global__ void __launch_bounds__(256) sort_clear_kernel(uint4* p, int64_t n) {
  follow();
  const int64_t i = blockIdx.x * 256LL + threadIdx.x;
  if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}

// ---- host ----------------------------------------------------------------------------------------
struct SortShape {
  int passes, bits, bins;
  bool team;  // sorted by one cluster
  int lists;  // lists between passes
  int64_t chunk, chunks;
};
inline SortShape sort_shape(int64_t n, int64_t n_keys) {
  SortShape s;
  int width = 2;  // bits of the largest key (n_keys: masked); four bins at least
  while ((n_keys >> width) > 0) ++width;
  s.passes = (width + kSortMaxBits - 1) / kSortMaxBits;
  s.bits = (width + s.passes - 1) / s.passes;
  s.bins = 1 << s.bits;
  s.lists = s.passes > 2 ? 2 : s.passes - 1;
  s.team = n <= kTeamMost;
  const int64_t tiles = (n + kSortTile - 1) / kSortTile;
  s.chunk = (tiles + kSortMaxChunks - 1) / kSortMaxChunks * kSortTile;
  s.chunks = s.team ? 0 : (n + s.chunk - 1) / s.chunk;
  return s;
}
// scratch: the lists between passes, and a table of counts for each
inline int64_t sort_bytes(int64_t n, int64_t n_keys) {
  const SortShape s = sort_shape(n, n_keys);
  return s.lists * align256(n * static_cast<int64_t>(sizeof(Entry))) +
         align256(s.passes * s.chunks * s.bins * 4);
}

template <class I, class Out>
int sort_team(const FromIds<I>& ids, int64_t n, const Out& out, const SortShape& s, Entry** list,
              uint8_t* clear, int64_t n_clear, int32_t* counter, cudaStream_t st) {
  auto kernel = &sort_team_kernel<I, Out>;
  auto smem = [](int bins) {
    return bins * (2 * sizeof(int) + kTeamWarps * sizeof(uint16_t));
  };
  ensure_dyn_smem(reinterpret_cast<const void*>(kernel), smem(kSortMaxBins));
  const unsigned ctas = n <= kTeamThreads ? 1 : kTeamCtas;
  cudaLaunchAttribute how[2];
  how[0].id = cudaLaunchAttributeClusterDimension;
  how[0].val.clusterDim = {ctas, 1, 1};
  how[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  how[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas);
  config.blockDim = dim3(kTeamThreads);
  config.dynamicSmemBytes = smem(s.bins);
  config.stream = st;
  config.attrs = how;
  config.numAttrs = 2;
  const int chunk = static_cast<int>((n + ctas * 32 - 1) / (ctas * 32) * 32);
  cudaLaunchKernelEx(&config, kernel, ids, out, static_cast<int>(n), chunk, s.bits, s.passes,
                     list[0], list[1], clear, n_clear, counter);
  return launch_status();
}

// Sorts ids 0 .. n - 1 into `out`; zeroes clear[0 .. n_clear) (padded to 16) and *counter before
// any entry is placed.
template <class I, class Out>
int sort_ids(const IdKeys<I>& ids, int64_t n, const Out& out, uint8_t* clear, int64_t n_clear,
             int32_t* counter, unsigned char* ws, cudaStream_t st) {
  const SortShape s = sort_shape(n, ids.n_keys);
  const FromIds<I> from_ids{ids};
  Entry* list[2] = {nullptr, nullptr};
  for (int b = 0; b < s.lists; ++b) {
    list[b] = reinterpret_cast<Entry*>(ws);
    ws += align256(n * static_cast<int64_t>(sizeof(Entry)));
  }
  if (s.team) {
    if (n_clear > (n <= kFewMost ? 1 << 17 : 1 << 20)) {
      const int64_t words = (n_clear + 15) / 16;
      const int status = launch_behind(&sort_clear_kernel,
                                       dim3(static_cast<unsigned>((words + 255) / 256)), 256, 0, st,
                                       reinterpret_cast<uint4*>(clear), words);
      if (status != B2S_OK) return status;
      n_clear = 0;
    }
    if constexpr (!Out::kOnePass) {
      if (n <= kFewMost)
        return launch_behind(&sort_few_kernel<I, Out>, dim3(1), kFewMost, 0, st, from_ids, out, n,
                             clear, n_clear, counter);
    }
    return sort_team<I, Out>(from_ids, n, out, s, list, clear, n_clear, counter, st);
  }
  int* counts = reinterpret_cast<int*>(ws);
  const size_t smem = sort_smem(s.bins);
  const unsigned grid = static_cast<unsigned>(s.chunks);
  const int64_t table = s.chunks * s.bins;
  auto place = [&](const auto& from, const auto& to, int p) {
    auto kernel = &sort_place_kernel<std::decay_t<decltype(from)>, std::decay_t<decltype(to)>>;
    ensure_dyn_smem(reinterpret_cast<const void*>(kernel), sort_smem(kSortMaxBins));
    const NextCounts next{p + 1 < s.passes ? counts + (p + 1) * table : nullptr,
                          static_cast<unsigned>(s.chunk), (p + 1) * s.bits};
    return launch_behind(kernel, grid, kSortThreads, smem, st, from, to, n, s.chunk, p * s.bits,
                         s.bins, counts + p * table, next);
  };
  int status = launch_behind(&sort_count_kernel<I>, grid, kSortThreads, s.bins * sizeof(int), st,
                             from_ids, n, s.chunk, s.bins, s.passes, counts, clear, n_clear,
                             counter);
  if (status != B2S_OK) return status;
  if constexpr (Out::kOnePass) {
    status = place(from_ids, out, 0);
  } else {
    status = s.passes == 1 ? place(from_ids, out, 0) : place(from_ids, ListOut{list[0]}, 0);
    for (int p = 1; p < s.passes && status == B2S_OK; ++p) {
      const FromList from{(p & 1) ? list[0] : list[1]};
      status = p + 1 == s.passes ? place(from, out, p)
                                 : place(from, ListOut{(p & 1) ? list[1] : list[0]}, p);
    }
  }
  return status;
}

}  // namespace b2s
