// Drawing the next id behind filters, one thread-block cluster a row.
//
// Candidates are ordered by logit descending, equal logits by id.  Weights w_i = exp((l_i - max) / T).  Every filter keeps
// a prefix of that order: top-k its first k; min-p those with w_i >= min_p (the largest weight is 1); top-p the shortest
// prefix whose sum reaches top_p times the sum Z of what top-k left (at least one).  With K the sum of the shortest of the
// three, the answer is the first candidate whose running sum passes u * K.
//
// A weight is computed in 64 bits and held as a whole number of 2^-S (S = 62 - bits of the vocabulary, at most 50): sums of
// whole numbers have no order, so a row's answer depends on its own logits and settings alone, and they are exact where a
// 32-bit sum over 150,000 candidates would move the draw to a neighbour in every hundredth row of a flat distribution.
//
// The order is never made.  A row's logits are read once, into the shared memory of its cluster's blocks; what follows goes
// by narrowing down:
//   1. the largest logit, the smallest finite one;
//   2. how many candidates lie in each of 2,048 bins of equal width below the largest and, unless top-k keeps few, the sum of
//      their weights (shared-memory additions, a count and a low word a candidate, now and then a high word);
//   3. the first block adds the bins up: it knows the bin of every border (what top-k keeps, the nucleus, the draw) and the
//      exact sum in front of it.  Where all bins that can be kept fit a list (2,048 candidates: top-k of the usual sizes, the
//      nucleus of a confident model), they are fetched once and everything is decided there; else a border's bin is fetched
//      at a time;
//   4. a list of up to 256 is ranked by comparing all with all; of a longer one the place of a goal is found among 2,048 finer
//      bins, whose few candidates are then ranked;
//   5. bins of more than 2,048 candidates (equal or almost equal logits by the thousand) are told apart by the 64 bits of
//      (logit, id) themselves, 11 bits a pass over the row.
//
// Bound by the chain of these steps, not by a unit (8 rows of 151,936: 34 us for 4.9 MB, issue slots 43 % taken, memory 2 %; 64 rows
// of 152,064: 92 us, 50 %, 5 %; one row behind top-k 20: 16.3 us, of which load 2.2, counts 3.6, adding up 2.6, fetch 2.1).
#include "common.cuh"

#define FS_THREADS 1024
#define FS_WARPS (FS_THREADS / 32)
#define FS_BINS 2048
#define FS_LIST 2048
#define FS_EACH 2                    // bins of a thread, and candidates of the list
#define FS_FEW 256                   // candidates that are ranked by comparing all with all
#define FS_MAX_CLUSTER 8
static_assert(FS_BINS == FS_THREADS * FS_EACH && FS_LIST == FS_BINS, "a thread has two bins and two candidates of the list");

typedef unsigned long long u64;

enum : int { FS_COUNTS = 1, FS_SUMS = 2, FS_RADIX = 3, FS_FETCH = 4, FS_FETCH_ORDER = 5 };

// What the blocks of a cluster do next: count the candidates of all bins, count them and add up their weights, cut the candidates
// whose place in the order lies in low..high by `shift`, fetch the candidates of bins first..last into the first block's list,
// or those whose place lies in low..high.
struct __align__(16) FsCommand {
  int what, first, last, shift;
  u64 low, high;
  int is_first, is_last, unused[2];  // nothing was asked in front of this, nothing is behind it
};

struct __align__(16) FsStats { float max, min; int odd, unused; };       // odd: a NaN or +infinity

__device__ __forceinline__ unsigned fs_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned fs_size() { unsigned r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void fs_arrive() {
  __syncwarp();                      // the barrier wants a warp whole, whatever loop it comes from
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void fs_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void fs_sync() { fs_arrive(); fs_wait(); }
__device__ __forceinline__ unsigned fs_peer(const void* local, unsigned rank) {
  unsigned theirs;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
  return theirs;
}
__device__ __forceinline__ unsigned fs_load32(const void* local, unsigned rank) {      // no memory clobber: several may be on their way
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(fs_peer(local, rank)));
  return v;
}
__device__ __forceinline__ void fs_store32(const void* local, unsigned rank, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(fs_peer(local, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void fs_store128(const void* local, unsigned rank, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};"
               ::"r"(fs_peer(local, rank)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void fs_store64(const void* local, unsigned rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(fs_peer(local, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned fs_add32(const void* local, unsigned rank, unsigned v) {
  unsigned old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(fs_peer(local, rank)), "r"(v) : "memory");
  return old;
}

// a larger value comes first; the lower id among equal ones (-0 and 0 are equal logits)
__device__ __forceinline__ unsigned fs_key(float v) {
  const unsigned b = __float_as_uint(v + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float fs_value(unsigned key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }
__device__ __forceinline__ u64 fs_order(float v, int id) { return (u64)fs_key(v) << 32 | (unsigned)~id; }

// What a row's weights need: t = (l - max) log2(e) / T, 2^t as 2^(n / 1,024) from a table times the series of 2^r, |r| <=
// 1 / 2,048, to its square (what is left out is below 2^-37 of a weight, a hundredth of what moves a draw among 150,000 equal
// candidates), rounded to a whole number of 2^-S.  With a table of 64 and the fifth power, pass 2 of 8 rows of 152,000 took 9.7 us
// instead of 8.9.
#define FS_TABLE 1024
struct FsWeight {
  double max, rate, least, unit;
  const double* table;      // 2^(j / FS_TABLE)
  __device__ __forceinline__ double plain(float l) const {
    const double t = ((double)l - max) * rate;
    if (!(t > least)) return 0.0;                 // below half a unit; a NaN (0 times infinity) too
    constexpr double kRound = 6755399441055744.0; // 1.5 * 2^52: adding it rounds to whole numbers
    constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2;
    const double n = fma(t, (double)FS_TABLE, kRound);
    const int whole = __double2loint(n);
    const double r = fma(n - kRound, -1.0 / FS_TABLE, t);
    const double v = table[whole & (FS_TABLE - 1)] * fma(r, fma(r, c2, c1), 1.0);
    return __hiloint2double(__double2hiint(v) + (whole >> 10) * (1 << 20), __double2loint(v));
  }
  __device__ __forceinline__ u64 whole(double w) const {        // w <= 1, unit <= 2^50
    return (u64)__double_as_longlong(fma(w, unit, 4503599627370496.0)) & ((1ull << 52) - 1);
  }
  __device__ __forceinline__ u64 operator()(float l) const { return whole(plain(l)); }
};

// how far a range of the order is shifted to leave fewer than FS_BINS parts
__device__ __forceinline__ int fs_shift(u64 range) { return max(0, 53 - __clzll((long long)range)); }

struct FsShared {
  u64 list[FS_LIST];                 // candidates; the sums of bins take the same place, low words and high words
  unsigned count[FS_BINS];
  unsigned all_count[FS_BINS];       // the first block's: counts and sums of the whole row
  u64 all_sum[FS_BINS];
  FsCommand command;
  FsStats stats[FS_MAX_CLUSTER];     // of the cluster's blocks, each written by its block
  uint4 ids[FS_MAX_CLUSTER];         // the first block's: the first id with the largest logit in each block's slice (x)
  ulonglong2 sums[FS_MAX_CLUSTER];   // the first block's: the weights above min-p's border in each block's slice (x)
  u64 scratch[2][2 * FS_WARPS];      // taken in turn, so that one barrier an exchange is enough
  double table[FS_TABLE];
  float of_warps[3][FS_WARPS];
  unsigned listed, mine;
  int first_id;
};

// Exchanges between a block's threads, each with one barrier: a buffer is written again two exchanges later, behind the barrier
// of the one between.
struct FsBlock {
  FsShared& sh;
  int turn;
  __device__ __forceinline__ u64* next() { turn ^= 1; return sh.scratch[turn]; }
  __device__ __forceinline__ u64 sum(u64 v) {                        // of all threads; every thread has it
    u64* at = next();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    v = at[threadIdx.x & (FS_WARPS - 1)];
#pragma unroll
    for (int o = FS_WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  __device__ __forceinline__ unsigned min(unsigned v) {
    unsigned* at = reinterpret_cast<unsigned*>(next());
    v = __reduce_min_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_min_sync(0xffffffffu, at[threadIdx.x & (FS_WARPS - 1)]);
  }
  // the one thread's values whose test holds
  __device__ __forceinline__ ulonglong2 from(bool mine, u64 v, u64 w = 0) {
    u64* at = next();
    if (mine) { at[0] = v; at[1] = w; }
    __syncthreads();
    return make_ulonglong2(at[0], at[1]);
  }
  // the count and the sum of the threads in front of this one, added to `count` and `sum`
  __device__ __forceinline__ void before(unsigned n, u64 v, unsigned& count, u64& sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64* at_v = next();
    unsigned* at_n = reinterpret_cast<unsigned*>(at_v + FS_WARPS);
    unsigned to_n = n;
    u64 to_v = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned un = __shfl_up_sync(0xffffffffu, to_n, o);
      const u64 uv = __shfl_up_sync(0xffffffffu, to_v, o);
      if (lane >= o) { to_n += un; to_v += uv; }
    }
    if (lane == 31) { at_n[warp] = to_n; at_v[warp] = to_v; }
    __syncthreads();
    // the warps in front: a lane each
    unsigned front_n = lane < warp ? at_n[lane & (FS_WARPS - 1)] : 0;
    u64 front_v = lane < warp ? at_v[lane & (FS_WARPS - 1)] : 0;
    front_n = __reduce_add_sync(0xffffffffu, front_n);
#pragma unroll
    for (int o = FS_WARPS / 2; o > 0; o >>= 1) front_v += __shfl_xor_sync(0xffffffffu, front_v, o);
    front_v = __shfl_sync(0xffffffffu, front_v, 0);
    count += front_n + to_n - n;
    sum += front_v + to_v - v;
  }
};

__global__ void __launch_bounds__(FS_THREADS, 1)
sample_filtered_kernel(const float* __restrict__ logits, int vocab, int slice, int resident, int unit_bits,
                       const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
                       const float* __restrict__ min_p, const float* __restrict__ uniform, int* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char fs_raw[];
  FsShared& sh = *reinterpret_cast<FsShared*>(fs_raw);
  float4* held = reinterpret_cast<float4*>(fs_raw + sizeof(FsShared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const unsigned rank = fs_rank(), size = fs_size();
  fs_arrive();                                   // every block runs before one writes into another: waited for further down
  const int row = blockIdx.x / size;
  const int begin = (int)min((long long)vocab, (long long)rank * slice), n = min(slice, vocab - begin);
  // The slice in groups of four that lie on 16 bytes; what of the first and the last group is not the slice's counts as -infinity.
  const float* global = logits + (size_t)row * vocab + begin;
  const int skew = (int)((reinterpret_cast<uintptr_t>(global) >> 2) & 3), groups = n > 0 ? (skew + n + 3) / 4 : 0;
  auto fetch4 = [&](int i) {
    const int at = 4 * i - skew;
    if (at >= 0 && at + 4 <= n) return *reinterpret_cast<const float4*>(global + at);
    float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (at >= 0 && at < n) v.x = global[at];
    if (at + 1 >= 0 && at + 1 < n) v.y = global[at + 1];
    if (at + 2 >= 0 && at + 2 < n) v.z = global[at + 2];
    if (at + 3 >= 0 && at + 3 < n) v.w = global[at + 3];
    return v;
  };
  auto group_of = [&](int i) { return resident ? held[i] : fetch4(i); };
  auto id_of = [&](int i, int e) { return begin + 4 * i - skew + e; };
  unsigned* low_word = reinterpret_cast<unsigned*>(sh.list);
  unsigned* high_word = low_word + FS_BINS;
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) sh.count[tid + i * FS_THREADS] = low_word[tid + i * FS_THREADS] = high_word[tid + i * FS_THREADS] = 0;
  };
  clear();
  static_assert(FS_TABLE == FS_THREADS, "a thread an entry");
  sh.table[tid] = exp2(tid / (double)FS_TABLE);
  if (tid == 0) { sh.listed = 0; sh.mine = 0; sh.first_id = 0x7fffffff; }
  pdl_wait();
  pdl_launch();
  const float temp = temperature[row];
  const int k_asked = top_k ? top_k[row] : 0;
  const float p_asked = top_p ? top_p[row] : 1.f, m_asked = min_p ? min_p[row] : 0.f, u_asked = uniform[row];

  // ---- 1. the slice into shared memory; its largest, smallest finite, and odd values ----
  FsStats all{-INFINITY, INFINITY, 0, 0};
  {
    constexpr int kAhead = 5;
    for (int i0 = tid; i0 < groups; i0 += kAhead * FS_THREADS) {
      float4 v[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        v[e] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i0 + e * FS_THREADS < groups) v[e] = fetch4(i0 + e * FS_THREADS);
      }
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        if (resident && i0 + e * FS_THREADS < groups) held[i0 + e * FS_THREADS] = v[e];
        const float x[4] = {v[e].x, v[e].y, v[e].z, v[e].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          all.max = fmaxf(all.max, x[c]);
          all.min = fminf(all.min, x[c] > -INFINITY ? x[c] : INFINITY);
          all.odd |= !(x[c] < INFINITY);
        }
      }
    }
  }
  auto join = [](FsStats& a, float max, float min, int odd) {
    a.max = fmaxf(a.max, max);
    a.min = fminf(a.min, min);
    a.odd |= odd;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    join(all, __shfl_xor_sync(0xffffffffu, all.max, o), __shfl_xor_sync(0xffffffffu, all.min, o), __shfl_xor_sync(0xffffffffu, all.odd, o));
  if (lane == 0) { sh.of_warps[0][warp] = all.max; sh.of_warps[1][warp] = all.min; sh.of_warps[2][warp] = __int_as_float(all.odd); }
  __syncthreads();
  fs_wait();
  if (warp == 0) {
    const int w = lane & (FS_WARPS - 1);
    all = FsStats{sh.of_warps[0][w], sh.of_warps[1][w], __float_as_int(sh.of_warps[2][w]), 0};
#pragma unroll
    for (int o = FS_WARPS / 2; o > 0; o >>= 1)
      join(all, __shfl_xor_sync(0xffffffffu, all.max, o), __shfl_xor_sync(0xffffffffu, all.min, o), __shfl_xor_sync(0xffffffffu, all.odd, o));
    if (lane < (int)size)
      fs_store128(&sh.stats[rank], lane, make_uint4(__float_as_uint(all.max), __float_as_uint(all.min), (unsigned)all.odd, 0u));
  }
  fs_sync();
  all = FsStats{-INFINITY, INFINITY, 0, 0};
  for (unsigned r = 0; r < size; ++r) join(all, sh.stats[r].max, sh.stats[r].min, sh.stats[r].odd);
  // greedy rows; rows whose weights have no finite sum; rows without a candidate
  if (!(temp > 0.f) || all.odd || all.max == -INFINITY) {
    if (all.max > -INFINITY) {
      int id = 0x7fffffff;
      for (int i = tid; i < groups; i += FS_THREADS) {
        const float4 v = group_of(i);
        if (v.w == all.max) id = min(id, id_of(i, 3));
        if (v.z == all.max) id = min(id, id_of(i, 2));
        if (v.y == all.max) id = min(id, id_of(i, 1));
        if (v.x == all.max) id = min(id, id_of(i, 0));
      }
      id = __reduce_min_sync(0xffffffffu, id);
      if (lane == 0) atomicMin(&sh.first_id, id);
      __syncthreads();
      if (tid == 0) fs_store128(&sh.ids[rank], 0, make_uint4((unsigned)sh.first_id, 0u, 0u, 0u));
      fs_sync();
      if (rank == 0 && tid == 0) {
        for (unsigned r = 0; r < size; ++r) id = min(id, (int)sh.ids[r].x);
        out[row] = id;
      }
    } else if (rank == 0 && tid == 0) {
      out[row] = 0;
    }
    return;
  }

  // ---- 2. the bins ----
  const double rate = 1.4426950408889634074 / (double)temp;       // log2(e) / T
  const FsWeight weight{(double)all.max, rate, -(double)(unit_bits + 1), (double)(1ull << unit_bits), sh.table};
  const float reach = fminf(all.max - all.min, (float)((unit_bits + 2) / rate));     // further down every weight is nothing
  const float bin_scale = reach > 0.f ? 2047.96875f / reach : 0.f;
  auto place_of = [&](float l) { return (all.max - l) * bin_scale; };                 // falls as l grows, as rounded too
  auto bin_of = [&](float x) { return min(FS_BINS - 1, (int)x); };                    // a NaN (0 times infinity): 0
  const bool by_k = k_asked > 0 && k_asked < vocab;
  const bool by_m = m_asked > 0.f, by_p = p_asked < 1.f;
  const double m_border = fmin((double)m_asked, 1.0), p_share = fmax((double)p_asked, 0.0);
  FsBlock block{sh, 0};
  // top-k of few: the bins' counts alone say what to fetch
  const bool count_only = by_k && k_asked <= FS_LIST / 2;
  auto add_to = [&](int at, u64 w) {
    const unsigned low = (unsigned)w, old = atomicAdd(&low_word[at], low);
    const unsigned high = (unsigned)(w >> 32) + (old + low < old);
    if (high) atomicAdd(&high_word[at], high);
  };
  // counts of the bins and, with `sums`, their weights and the sum of those above min-p's border (told to the first block)
  auto add_bins = [&](bool sums) {
    u64 m_sum = 0;
    for (int i = tid; i < groups; i += FS_THREADS) {
      const float4 v = group_of(i);
      const float x[4] = {v.x, v.y, v.z, v.w};
      int at[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        at[c] = bin_of(place_of(x[c]));
        if (x[c] > -INFINITY) atomicAdd(&sh.count[at[c]], 1u);
      }
      if (sums) {
        double w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = weight.plain(x[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const u64 whole = weight.whole(w[c]);
          if (whole) add_to(at[c], whole);
          if (by_m && w[c] >= m_border) m_sum += whole;
        }
      }
    }
    if (sums && by_m) {
      m_sum = block.sum(m_sum);
      if (tid == 0) fs_store128(&sh.sums[rank], 0, make_uint4((unsigned)m_sum, (unsigned)(m_sum >> 32), 0u, 0u));
    }
  };
  // ---- what the first block asks for, by all blocks ----
  auto serve = [&](const FsCommand& c) {
    if (c.what <= FS_RADIX) {
      if (!c.is_first) {                           // they are clear; the first block has what they were in its threads' registers
        clear();
        __syncthreads();
      }
      if (c.what <= FS_SUMS) {
        add_bins(c.what == FS_SUMS);
        return;
      }
    } else {
      if (tid == 0) sh.mine = 0;
      __syncthreads();
    }
    auto take = [&](float l, int id) {
      const unsigned to = atomicAdd(rank == 0 ? &sh.listed : &sh.mine, 1u);
      if (to < FS_LIST) sh.list[to] = fs_order(l, id);
    };
    if (c.what == FS_FETCH) {
      // a place lies in bins first..last where first <= place < last + 1 (the last bin has no end: nothing is >= a NaN; a place that
      // is a NaN lies in bin 0)
      const float low = (float)c.first, high = c.last < FS_BINS - 1 ? (float)(c.last + 1) : __int_as_float(0x7fc00000);
      const bool from_top = c.first == 0;
      for (int i = tid; i < groups; i += FS_THREADS) {
        const float4 v = group_of(i);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = place_of(x[e]);
          if (x[e] > -INFINITY && (from_top || p >= low) && !(p >= high)) take(x[e], id_of(i, e));
        }
      }
    } else {
      for (int i = tid; i < groups; i += FS_THREADS) {
        const float4 v = group_of(i);
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const float l = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
          const u64 order = fs_order(l, id_of(i, e));
          if (!(l > -INFINITY) || order < c.low || order > c.high) continue;
          if (c.what == FS_RADIX) {
            const int at = (int)((c.high - order) >> c.shift);
            atomicAdd(&sh.count[at], 1u);
            add_to(at, weight(l));
          } else {
            take(l, id_of(i, e));
          }
        }
      }
    }
    if (c.what != FS_RADIX && rank != 0) {
      __syncthreads();
      const unsigned mine = min(sh.mine, (unsigned)FS_LIST);
      if (mine) {                                  // the same for the block
        const u64 base = block.from(tid == 0, tid == 0 ? fs_add32(&sh.listed, 0, mine) : 0u).x;
        for (unsigned i = tid; i < mine; i += FS_THREADS)
          if (base + i < FS_LIST) fs_store64(&sh.list[base + i], 0, sh.list[i]);
      }
    }
  };
  // What has been cut, added up over the cluster into the first block's shared memory: a block has every size-th part of the
  // bins, a thread two blocks' counts and sums of one (the first block alone, reading them all one behind the other, took
  // 13.5 us for counts and sums of 8 blocks and what follows from them, this 3.6).
  auto gather = [&](bool sums) {
    const int halves = size / 2, bin = rank * (FS_BINS / size) + tid / halves, r = tid % halves * 2;
    unsigned n = fs_load32(&sh.count[bin], r) + fs_load32(&sh.count[bin], r + 1);
    u64 v = 0;
    if (sums) {
      const unsigned low0 = fs_load32(low_word + bin, r), low1 = fs_load32(low_word + bin, r + 1);
      const unsigned high0 = fs_load32(high_word + bin, r), high1 = fs_load32(high_word + bin, r + 1);
      v = (u64)low0 + low1 + ((u64)(high0 + high1) << 32);
    }
    for (int o = 1; o < halves; o <<= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, o);
      v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    if (r == 0) {
      fs_store32(&sh.all_count[bin], 0, n);
      if (sums) fs_store64(&sh.all_sum[bin], 0, v);
    }
  };
  // the thread's bins of that (or of this block's own), and running ones behind `n_front` candidates of sum `front`
  unsigned count_of[FS_EACH] = {}, count_to[FS_EACH] = {};
  u64 sum_to[FS_EACH] = {};
  auto add_up = [&](bool own, bool sums, unsigned n_front, u64 front, unsigned (&of)[FS_EACH], unsigned (&to)[FS_EACH], u64 (&sum)[FS_EACH]) {
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) {
      const int at = tid * FS_EACH + i;
      of[i] = own ? sh.count[at] : sh.all_count[at];
      sum[i] = !sums ? 0 : own ? low_word[at] + ((u64)high_word[at] << 32) : sh.all_sum[at];
    }
    to[0] = of[0];
#pragma unroll
    for (int i = 1; i < FS_EACH; ++i) { to[i] = to[i - 1] + of[i]; sum[i] += sum[i - 1]; }
    block.before(to[FS_EACH - 1], sum[FS_EACH - 1], n_front, front);
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) { to[i] += n_front; sum[i] += front; }
  };
  // the first of all places (a thread has FS_EACH) whose test holds; FS_BINS if none does
  auto first_of = [&](auto holds) {
    unsigned at = FS_BINS;
#pragma unroll
    for (int i = FS_EACH - 1; i >= 0; --i)
      if (holds(i)) at = tid * FS_EACH + i;
    return (int)block.min(at);
  };
  // of numbers that the threads have FS_EACH of, the one at a place
  auto at_place = [&](const auto& v, int b) {
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i)
      if ((b & (FS_EACH - 1)) == i) mine = (u64)v[i];
    return block.from(tid == b / FS_EACH, mine).x;
  };
  // what bin b holds: its count, and count and sum of what lies in front of it
  struct Bin { unsigned here, count; u64 sum; };
  auto bin_at = [&](const unsigned (&of)[FS_EACH], const unsigned (&to)[FS_EACH], const u64 (&sum)[FS_EACH], int b, u64 none) {
    const bool mine = tid == b / FS_EACH, before = tid == (b - 1) / FS_EACH && b > 0;
    u64* at = block.next();
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) {
      if (mine && (b & (FS_EACH - 1)) == i) at[0] = (u64)(to[i] - of[i]) << 32 | of[i];
      if (before && ((b - 1) & (FS_EACH - 1)) == i) at[1] = sum[i];
    }
    __syncthreads();
    return Bin{(unsigned)at[0], (unsigned)(at[0] >> 32), b > 0 ? at[1] : none};
  };

  // A goal: the goal-th candidate of the order (by_count), or the first whose running sum is > goal (strict) or >= goal.
  struct Goal {
    bool by_count, strict;
    double goal;
    __device__ __forceinline__ bool reached(unsigned count, u64 sum) const {
      return by_count ? (double)count >= goal : strict ? (double)sum > goal : (double)sum >= goal;
    }
  };
  struct Found { u64 sum, order; };              // the running sum at the candidate, its place in the order

  // ---- 4. the list: in threads' registers, with weights; behind `n_front` candidates of sum `front` ----
  u64 order_at[FS_EACH], weight_at[FS_EACH];
  int in_list = 0;
  unsigned n_front = 0, rank_at = 0;
  u64 front = 0, ranked_sum = 0, ranked = 0;     // of a list of few: this thread's candidate, its rank, the running sum there
  // ranks of the first n candidates in sh.list, weights behind them at FS_FEW: four threads a candidate, each compares it with
  // every fourth (one thread a candidate took 7.4 us for 250, this 3.5)
  static_assert(FS_THREADS == 4 * FS_FEW, "four threads a candidate");
  auto ranks_here = [&](int n) { return (tid & 3) == 0 && tid / 4 < n; };
  auto rank_few = [&](int n, unsigned count, u64 sum) {
    ranked = tid / 4 < n ? sh.list[tid / 4] : ~0ull;
    rank_at = 0;
    ranked_sum = 0;
    if (warp * 8 < n) {
#pragma unroll 4
      for (int j = tid & 3; j < n; j += 4) {
        const u64 other = sh.list[j], w = sh.list[FS_FEW + j];
        if (other >= ranked) { ++rank_at; ranked_sum += w; }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        rank_at += __shfl_xor_sync(0xffffffffu, rank_at, o);
        ranked_sum += __shfl_xor_sync(0xffffffffu, ranked_sum, o);
      }
    }
    rank_at += count;
    ranked_sum += sum;
  };
  // among n ranked ones behind `count` others (where none reaches the goal: the last one)
  auto first_ranked = [&](int n, unsigned count, const Goal& goal) {
    const unsigned at = min(block.min(ranks_here(n) && goal.reached(rank_at, ranked_sum) ? rank_at : 0xffffffffu), count + n);
    const ulonglong2 found = block.from(ranks_here(n) && rank_at == at, ranked_sum, ranked);
    return Found{found.x, found.y};
  };
  // a longer one: cut into 2,048 parts of its order (or of low..high of it, behind `count` candidates of sum `sum`)
  unsigned list_of[FS_EACH], list_to[FS_EACH];
  u64 list_sum[FS_EACH], least = 0, most = 0, cut_low = 0, cut_high = 0, cut_sum = 0;
  int cut_shift = 0;
  auto cut_list = [&](u64 low, u64 high, unsigned count, u64 sum) {
    cut_low = low;
    cut_high = high;
    cut_sum = sum;
    cut_shift = fs_shift(high - low);
    __syncthreads();
    clear();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i)
      if (tid + i * FS_THREADS < in_list && order_at[i] >= low && order_at[i] <= high) {
        const int at = (int)((high - order_at[i]) >> cut_shift);
        atomicAdd(&sh.count[at], 1u);
        add_to(at, weight_at[i]);
      }
    __syncthreads();
    add_up(true, true, count, sum, list_of, list_to, list_sum);
  };
  auto open_list = [&](unsigned count, u64 sum) {
    in_list = min((int)sh.listed, FS_LIST);
    n_front = count;
    front = sum;
    unsigned low = 0xffffffffu, high = 0xffffffffu;                          // keys, the second from above
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) {
      const int at = tid + i * FS_THREADS;
      order_at[i] = weight_at[i] = 0;
      if (at < in_list) {
        order_at[i] = sh.list[at];
        const unsigned key = (unsigned)(order_at[i] >> 32);
        weight_at[i] = weight(fs_value(key));
        low = min(low, key);
        high = min(high, ~key);
      }
    }
    if (in_list <= FS_FEW) {
      if (tid < in_list) sh.list[FS_FEW + tid] = weight_at[0];
      __syncthreads();
      rank_few(in_list, n_front, front);
    } else {
      least = (u64)block.min(low) << 32;
      most = (u64)~block.min(high) << 32 | 0xffffffffu;
      cut_list(least, most, n_front, front);
    }
  };
  auto find_in_list = [&](const Goal& goal) {
    if (in_list <= FS_FEW) return first_ranked(in_list, n_front, goal);
    if (cut_low != least || cut_high != most) cut_list(least, most, n_front, front);
    while (true) {
      const int at = first_of([&](int i) { return list_of[i] > 0 && goal.reached(list_to[i], list_sum[i]); });
      // a nucleus that ends behind what min-p keeps: all of the list
      if (at >= FS_BINS) return Found{at_place(list_sum, FS_BINS - 1), 0};
      const Bin bin = bin_at(list_of, list_to, list_sum, at, cut_sum);
      const u64 high = cut_high - ((u64)at << cut_shift), span = (1ull << cut_shift) - 1;
      const u64 low = high - cut_low > span ? high - span : cut_low;
      if (bin.here <= FS_FEW) {
        if (tid == 0) sh.mine = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FS_EACH; ++i)
          if (tid + i * FS_THREADS < in_list && order_at[i] >= low && order_at[i] <= high) {
            const unsigned to = atomicAdd(&sh.mine, 1u);
            sh.list[to] = order_at[i];
            sh.list[FS_FEW + to] = weight_at[i];
          }
        __syncthreads();
        rank_few((int)bin.here, bin.count, bin.sum);
        return first_ranked((int)bin.here, bin.count, goal);
      }
      cut_list(low, high, bin.count, bin.sum);
    }
  };

  // ---- 3 and 5. the first block decides what comes next, until the draw is found ----
  const double u = u_asked >= 0.f ? fmin((double)u_asked, 1.0 - 1.0 / 16777216) : 0.0;
  // An edge's weight from the single-precision exponential is off by less than 2^-16 of itself at the exponents that count, what
  // a place is rounded by included.
  const float step_log2 = bin_scale > 0.f ? (float)(1.0 / (double)bin_scale * rate) : 0.f;
  enum : int { kTopK, kNucleus, kDraw };
  int step = kTopK, end = 0, cut_by = 0;         // cut_by: what the threads' counts and sums are of (0: of nothing that serves)
  bool listed = false, open = false, k_cuts = false;
  unsigned count = 0;                            // in front of what was asked for, and their sum
  u64 sum = 0, kept = 0;                         // the sum of what is kept so far
  Goal k_goal{true, false, 0.0};
  // A list of up to 64 holds all that can be kept (top-k of the usual sizes): one warp decides, two candidates a lane, without an
  // exchange with the others (1 row, top-k 20 with top-p and min-p: 19.0 us with them, 16.2 without).
  auto draw_from_few = [&]() {
    if (warp != 0) return;
    const int n = (int)sh.listed;
    u64 order[2], at_sum[2] = {0, 0};
    unsigned at_rank[2] = {0, 0};
    double w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      order[e] = lane + 32 * e < n ? sh.list[lane + 32 * e] : ~0ull;
      w[e] = lane + 32 * e < n ? weight.plain(fs_value((unsigned)(order[e] >> 32))) : 0.0;
      if (lane + 32 * e < n) sh.list[FS_FEW + lane + 32 * e] = weight.whole(w[e]);
    }
    __syncwarp();
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 other = sh.list[j], whole = sh.list[FS_FEW + j];
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (other >= order[e]) { ++at_rank[e]; at_sum[e] += whole; }
    }
    auto first = [&](const Goal& goal) {
      unsigned at = n;                             // none reaches it: the last one
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lane + 32 * e < n && goal.reached(at_rank[e], at_sum[e])) at = min(at, at_rank[e]);
      at = __reduce_min_sync(0xffffffffu, at);
      const unsigned in0 = __ballot_sync(0xffffffffu, lane < n && at_rank[0] == at);
      const unsigned in1 = __ballot_sync(0xffffffffu, lane + 32 < n && at_rank[1] == at);
      const int from = __ffs(in0 ? in0 : in1) - 1;
      return Found{__shfl_sync(0xffffffffu, in0 ? at_sum[0] : at_sum[1], from), __shfl_sync(0xffffffffu, in0 ? order[0] : order[1], from)};
    };
    if (by_k) kept = first(k_goal).sum;
    if (by_p) kept = min(kept, first(Goal{false, false, p_share * (double)kept}).sum);
    if (by_m) {
      u64 m_sum = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lane + 32 * e < n && w[e] >= m_border) m_sum += weight.whole(w[e]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m_sum += __shfl_xor_sync(0xffffffffu, m_sum, o);
      kept = min(kept, m_sum);
    }
    const Found drawn = first(Goal{false, true, u * (double)kept});
    if (lane == 0) out[row] = (int)~(unsigned)drawn.order;
  };
  FsCommand c{};
  c.what = count_only ? FS_COUNTS : FS_SUMS;
  c.is_first = 1;
  while (true) {
    serve(c);
    fs_sync();                                   // it has been carried out
    if (c.what <= FS_RADIX && size > 1) {
      gather(c.what != FS_COUNTS);
      fs_sync();
    }
    if (rank != 0) {
      if (c.is_last) return;
      fs_sync();                                 // a command is there
      c = sh.command;
      continue;
    }
    if (c.what <= FS_RADIX) {
      add_up(size == 1, c.what != FS_COUNTS, count, sum, count_of, count_to, sum_to);
      cut_by = c.what;
      if (c.is_first) {
        const unsigned candidates = (unsigned)at_place(count_to, FS_BINS - 1);
        k_cuts = by_k && (unsigned)k_asked < candidates;
        k_goal.goal = (double)(k_cuts ? (unsigned)k_asked : candidates);
        if (!count_only) kept = at_place(sum_to, FS_BINS - 1);
        // the last bin that can hold a kept candidate: top-k's, the nucleus' (where what it is a share of is known), min-p's (where
        // nothing behind it is needed), the last one; and whether all up to it fit the list
        const double p_goal = p_share * (double)kept;
        end = first_of([&](int i) {
          return k_goal.reached(count_to[i], 0) || (by_p && !by_k && (double)sum_to[i] >= p_goal) ||
                 (by_m && !(by_k && by_p) && (double)exp2f(-(float)(tid * FS_EACH + i + 1) * step_log2) * (1 + 1.0 / 16384) < m_border);
        });
        listed = at_place(count_to, end) <= FS_LIST;
      }
    } else if (listed && sh.listed <= 64) {
      draw_from_few();
      return;
    } else {
      open_list(count, sum);
      open = true;
    }
    while (true) {
      if ((step == kTopK && !(listed ? by_k : k_cuts)) || (step == kNucleus && !by_p)) { ++step; continue; }
      if (step == kDraw && by_m && (open || !listed)) {
        u64 m_sum = 0;
        if (listed) {
#pragma unroll
          for (int i = 0; i < FS_EACH; ++i)
            if (tid + i * FS_THREADS < in_list && weight.plain(fs_value((unsigned)(order_at[i] >> 32))) >= m_border) m_sum += weight_at[i];
          m_sum = block.sum(m_sum);
        } else {
          for (unsigned r = 0; r < size; ++r) m_sum += sh.sums[r].x;
        }
        kept = min(kept, m_sum);
      }
      const Goal goal = step == kTopK ? k_goal : Goal{false, step == kDraw, (step == kDraw ? u : p_share) * (double)kept};
      if (open) {
        const Found found = find_in_list(goal);
        if (step == kDraw) {
          if (tid == 0) out[row] = (int)~(unsigned)found.order;
          return;
        }
        kept = step == kTopK ? found.sum : min(kept, found.sum);
        ++step;
        open = listed;
        if (cut_by == FS_RADIX) cut_by = 0;
        continue;
      }
      c.is_first = 0;
      c.is_last = listed || step == kDraw;
      if (listed) {
        c.what = FS_FETCH;
        c.first = 0;
        c.last = end;
        count = 0;
        sum = 0;
      } else if (cut_by != FS_SUMS && cut_by != FS_RADIX) {
        c.what = FS_SUMS;
        c.is_last = 0;
        count = 0;
        sum = 0;
      } else {
        const int at = min(FS_BINS - 1, first_of([&](int i) { return count_of[i] > 0 && goal.reached(count_to[i], sum_to[i]); }));
        const Bin bin = bin_at(count_of, count_to, sum_to, at, cut_by == FS_SUMS ? 0 : sum);
        count = bin.count;
        sum = bin.sum;
        if (cut_by == FS_RADIX) {
          const u64 span = (1ull << c.shift) - 1;
          c.high -= (u64)at << c.shift;
          c.low = c.high - c.low > span ? c.high - span : c.low;
          c.what = bin.here > FS_LIST ? FS_RADIX : FS_FETCH_ORDER;
        } else if (bin.here > FS_LIST) {             // from the whole order on
          c.what = FS_RADIX;
          c.low = (u64)fs_key(all.min) << 32;
          c.high = (u64)fs_key(all.max) << 32 | 0xffffffffu;
          count = 0;
          sum = 0;
        } else {
          c.what = FS_FETCH;
          c.first = c.last = at;
        }
        c.shift = fs_shift(c.high - c.low);
        if (c.what == FS_RADIX) c.is_last = 0;
      }
      break;
    }
    __syncthreads();
    if (warp == 0) {
      const uint4* words = reinterpret_cast<const uint4*>(&c);
      if (lane < (int)size)
        for (int i = 0; i < (int)(sizeof(FsCommand) / 16); ++i) fs_store128(reinterpret_cast<uint4*>(&sh.command) + i, lane, words[i]);
      if (lane == 0) sh.listed = 0;
    }
    fs_sync();
  }
}

// Blocks a cluster.  A block has a multiprocessor to itself, and the device holds some 16 clusters of 8 or 34 of 4 at once: few
// rows are cut into 8 slices, many into 2.  Slices below some 3,000 logits are not worth an exchange.  us for 8 / 4 / 2 / 1
// blocks, rows with settings of their own: 152,064 logits, 8 rows 39 / 53 / 89 / 151, 24 50 / 50 / 78 / 127, 64 103 / 91 / 124 / 206 (all
// from a nucleus 134 / 98 / 82 / 131); 49,999, 8 rows 31 / 35 / 43 / 66, 37 56 / 48 / 58 / 88, 64 77 / 52 / 58 / 89 (from a nucleus 93 / 57 /
// 38 / 56); 10,007, 37 rows 48 / 36 / 37 / 36; 2,000, 8 rows 20 / 19 / 19 / 18.  Which is faster goes by
// the settings too, and those are on the device: the rule bears its loss where they are of the other kind (64 rows of 152,064 from a
// nucleus 98 where 2 blocks take 82; of 49,999 with settings of their own 37 rows 58 where 4 take 48, 64 rows 58 where 4 take 52).
static int fs_cluster(int n_rows, int vocab) {
  const int by_rows = n_rows <= 15 ? 8 : n_rows <= (vocab > 100000 ? 68 : 34) ? 4 : 2;
  const int by_slice = vocab > 24576 ? 8 : vocab > 8192 ? 4 : vocab > 3000 ? 2 : 1;
  return by_rows < by_slice ? by_rows : by_slice;
}

// Draws one id a row of `logits` [n_rows][vocab].  `top_k` (0 or less: off), `top_p` (1 or more: off) and `min_p` (0: off) may be
// null; `uniform` holds numbers from [0, 1).
TOKB200_API int tokb200_sample_filtered(const float* logits, int n_rows, int vocab, const float* temperature, const int* top_k,
                                        const float* top_p, const float* min_p, const float* uniform, int* out,
                                        cudaStream_t stream) {
  if (n_rows <= 0) return TOKB200_OK;
  if (vocab <= 0 || n_rows > (1 << 27)) return TOKB200_BAD_SIZE;
  const int cluster = fs_cluster(n_rows, vocab);
  const int slice = (vocab + cluster - 1) / cluster;
  constexpr size_t kMost = 224 * 1024;               // of a block's shared memory
  const size_t held = ((size_t)slice + 8) * 4;       // in groups of four, of which the first and the last may be cut
  const bool resident = sizeof(FsShared) + held <= kMost;
  const size_t smem = sizeof(FsShared) + (resident ? held : 0);
  int bits = 0;
  while (((long long)1 << bits) < vocab) ++bits;
  const int unit_bits = 62 - bits < 50 ? 62 - bits : 50;
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return TOKB200_BAD_SIZE;
  if (!configured[device]) {
    cudaError_t err = cudaFuncSetAttribute(sample_filtered_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMost);
    if (err != cudaSuccess) return (int)err;
    configured[device] = true;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)n_rows * cluster);
  config.blockDim = dim3(FS_THREADS);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = tokb200_early_starts();
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = (unsigned)cluster;
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&config, sample_filtered_kernel, logits, vocab, slice, (int)resident, unit_bits,
                                             temperature, top_k, top_p, min_p, uniform, out);
  return err == cudaSuccess ? TOKB200_OK : (int)err;
}
