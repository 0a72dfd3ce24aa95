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
//   1. the largest logit, its lowest id (the greedy choice), the smallest finite one;
//   2. how many candidates lie in each of 2,048 bins of equal width below the largest (one shared-memory count a
//      candidate), and, unless top-k says what is summed, the sum of all weights;
//   3. the first block adds the bins up.  A bin's weights lie between those of its edges, so the counts alone bound every
//      running sum from both sides.  Where all that can be kept fits a list (2,048: top-k of the usual sizes, the nucleus
//      of a confident model) it is fetched, sorted, and everything is decided there;
//   4. else each border in turn (what top-k keeps, the nucleus, the draw): the bins that can hold it are fetched and
//      sorted, with the exact sum of what lies in front of them; where they hold more than the list, they are first cut
//      into 2,048 finer bins with exact sums;
//   5. candidates that finer bins cannot tell apart (equal or almost equal logits by the thousand) are told apart by the
//      64 bits of (logit, id) themselves, 11 bits a pass.
#include "common.cuh"

#define FS_THREADS 512
#define FS_WARPS (FS_THREADS / 32)
#define FS_BINS 2048
#define FS_LIST 2048
#define FS_EACH 4                    // bins of a thread, and places of the sorted list
#define FS_MAX_CLUSTER 8
static_assert(FS_BINS == FS_THREADS * FS_EACH && FS_LIST == FS_BINS, "a thread has four bins and four places of the list");

typedef unsigned long long u64;

enum : int { FS_FETCH = 1, FS_FINE = 2, FS_FETCH_FINE = 3, FS_RADIX = 4, FS_FETCH_ORDER = 5 };

// What the first block asks of the cluster: candidates of bins first..last (cut into finer bins with `fine_scale`, of which
// it may want `fine` alone), or those whose place in the order lies in low..high (cut by `shift`).
struct __align__(16) FsCommand {
  int what, first, last, fine;
  u64 low, high;
  int shift;
  float fine_scale;
  int want_front, want_m;            // the sum of what lies in front; the sum of the weights above min-p's border
  int is_last, unused[3];            // nothing is asked behind this
};

struct __align__(16) FsStats { float max, min; int odd, unused; };       // odd: a NaN or +infinity

__device__ __forceinline__ unsigned fs_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned fs_size() { unsigned r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void fs_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void fs_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void fs_sync() { fs_arrive(); fs_wait(); }
__device__ __forceinline__ unsigned fs_peer(const void* local, unsigned rank) {
  unsigned theirs;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
  return theirs;
}
__device__ __forceinline__ uint4 fs_load128(const void* local, unsigned rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(fs_peer(local, rank)) : "memory");
  return v;
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

// What a row's weights need: t = (l - max) log2(e) / T, 2^t as 2^(n / 64) from a table times the series of 2^r, |r| <=
// 1/128, to the fifth power (what is left out is below 2^-55), rounded to a whole number of 2^-S.
struct FsWeight {
  double max, rate, least, unit;
  const double* table;      // 2^(j / 64)
  __device__ __forceinline__ double plain(float l) const {
    const double t = ((double)l - max) * rate;
    if (!(t > least)) return 0.0;                 // below half a unit; a NaN (0 times infinity) too
    constexpr double kRound = 6755399441055744.0; // 1.5 * 2^52: adding it rounds to whole numbers
    constexpr double c1 = 0.69314718055994530942, c2 = c1 * c1 / 2, c3 = c2 * c1 / 3, c4 = c3 * c1 / 4, c5 = c4 * c1 / 5;
    const double n = fma(t, 64.0, kRound);
    const int whole = __double2loint(n);
    const double r = fma(n - kRound, -1.0 / 64, t);
    const double p = fma(r, fma(r, fma(r, fma(r, fma(r, c5, c4), c3), c2), c1), 1.0);
    const double v = table[whole & 63] * p;
    return __hiloint2double(__double2hiint(v) + (whole >> 6) * (1 << 20), __double2loint(v));
  }
  __device__ __forceinline__ u64 whole(double w) const {        // w <= 1, unit <= 2^50
    return (u64)__double_as_longlong(fma(w, unit, 4503599627370496.0)) & ((1ull << 52) - 1);
  }
  __device__ __forceinline__ u64 operator()(float l) const { return whole(plain(l)); }
};

struct FsShared {
  u64 list[FS_LIST];                 // candidates; the sums of finer bins take the same place, low words and high words
  unsigned count[FS_BINS];
  FsCommand command;
  FsStats stats[FS_MAX_CLUSTER];     // of the cluster's blocks, each written by its block
  uint4 ids[FS_MAX_CLUSTER];         // the first block's: the first id with the largest logit in each block's slice (x)
  ulonglong2 sums[FS_MAX_CLUSTER];   // the first block's: of each block all weights (or those in front), those above min-p's border
  u64 scratch[2][3 * FS_WARPS];      // taken in turn, so that one barrier an exchange is enough
  double table[64];
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
  // the one thread's value whose test holds
  __device__ __forceinline__ u64 from(bool mine, u64 v) {
    u64* at = next();
    if (mine) at[0] = v;
    __syncthreads();
    return at[0];
  }
  // sums of the threads in front of this one, of three numbers at once
  template <typename A, typename B, typename C>
  __device__ __forceinline__ void before(A& a, B& b, C& c) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64* at = next();
    A* at_a = reinterpret_cast<A*>(at);
    B* at_b = reinterpret_cast<B*>(at + FS_WARPS);
    C* at_c = reinterpret_cast<C*>(at + 2 * FS_WARPS);
    A sa = a; B sb = b; C sc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const A ua = __shfl_up_sync(0xffffffffu, sa, o);
      const B ub = __shfl_up_sync(0xffffffffu, sb, o);
      const C uc = __shfl_up_sync(0xffffffffu, sc, o);
      if (lane >= o) { sa += ua; sb += ub; sc += uc; }
    }
    if (lane == 31) { at_a[warp] = sa; at_b[warp] = sb; at_c[warp] = sc; }
    __syncthreads();
    A fa = 0; B fb = 0; C fc = 0;
    for (int w = 0; w < warp; ++w) { fa += at_a[w]; fb += at_b[w]; fc += at_c[w]; }
    a = fa + sa - a; b = fb + sb - b; c = fc + sc - c;
  }
};

// Descending order of FS_LIST numbers (or of the first `n`, a power of two from 128 on), four to a thread side by side: a warp's
// 128 exchange in registers, pairs further apart through `list`.
__device__ __forceinline__ void fs_sort(u64 (&v)[FS_EACH], u64* list, int n) {
  const int tid = threadIdx.x, base = tid * FS_EACH;
  auto keep = [](u64& a, u64& b, bool down) { if ((a < b) == down) { const u64 x = a; a = b; b = x; } };
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 128) {
        __syncthreads();
        if (base < n) {
#pragma unroll
          for (int i = 0; i < FS_EACH; ++i) list[base + i] = v[i];
        }
        __syncthreads();
        if (base < n) {
#pragma unroll
          for (int i = 0; i < FS_EACH; ++i) {
            const int at = base + i;
            const u64 other = list[at ^ j];
            const bool larger = ((at & k) == 0) == ((at & j) == 0);        // this place keeps the larger of the two
            if ((other > v[i]) == larger) v[i] = other;
          }
        }
      } else if (base < n) {                                              // whole warps
        if (j >= 4) {
#pragma unroll
          for (int i = 0; i < FS_EACH; ++i) {
            const u64 other = __shfl_xor_sync(0xffffffffu, v[i], j >> 2);
            const bool larger = (((base + i) & k) == 0) == (((base + i) & j) == 0);
            if ((other > v[i]) == larger) v[i] = other;
          }
        } else if (j == 2) {
          const bool down = (base & k) == 0;                              // k >= 4: the same for a thread's four
          keep(v[0], v[2], down);
          keep(v[1], v[3], down);
        } else {
          keep(v[0], v[1], (base & k) == 0);
          keep(v[2], v[3], ((base + 2) & k) == 0);
        }
      }
    }
}

__global__ void __launch_bounds__(FS_THREADS, 2)
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
#pragma unroll
  for (int i = 0; i < FS_EACH; ++i) sh.count[tid + i * FS_THREADS] = 0;
  if (tid < 64) sh.table[tid] = exp2(tid / 64.0);
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
  auto tell = [&](u64 a, u64 b) {                                 // the first block, of this one's sums
    fs_store128(&sh.sums[rank], 0, make_uint4((unsigned)a, (unsigned)(a >> 32), (unsigned)b, (unsigned)(b >> 32)));
  };
  {
    u64 sum = 0, m_sum = 0;
    for (int i = tid; i < groups; i += FS_THREADS) {
      const float4 v = group_of(i);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (x[c] > -INFINITY) atomicAdd(&sh.count[bin_of(place_of(x[c]))], 1u);
      if (!by_k) {
        double w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = weight.plain(x[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sum += weight.whole(w[c]);
          if (by_m && w[c] >= m_border) m_sum += weight.whole(w[c]);
        }
      }
    }
    if (!by_k) {
      sum = block.sum(sum);
      if (by_m) m_sum = block.sum(m_sum);
    }
    if (tid == 0) tell(sum, m_sum);
  }
  fs_sync();

  // ---- what the first block asks for, by all blocks: candidates into its list, or counts and sums of what is cut ----
  auto serve = [&](const FsCommand& c) {
    const bool cut = c.what == FS_FINE || c.what == FS_RADIX;
    u64 front = 0, m_sum = 0;
    unsigned* low_word = reinterpret_cast<unsigned*>(sh.list);
    unsigned* high_word = low_word + FS_BINS;
    if (cut) {
      // the first block has the counts of all bins in its threads' registers by now
#pragma unroll
      for (int i = 0; i < FS_EACH; ++i) sh.count[tid + i * FS_THREADS] = low_word[tid + i * FS_THREADS] = high_word[tid + i * FS_THREADS] = 0;
    }
    if (tid == 0) sh.mine = 0;
    __syncthreads();
    auto take = [&](float l, int id) {
      if (rank == 0) {
        const unsigned to = atomicAdd(&sh.listed, 1u);
        if (to < FS_LIST) sh.list[to] = fs_order(l, id);
      } else {
        const unsigned to = atomicAdd(&sh.mine, 1u);
        if (to < FS_LIST) sh.list[to] = fs_order(l, id);
      }
    };
    if (c.what == FS_FETCH) {
      // a place lies in bins first..last where first <= place < last + 1 (the last bin has no end: nothing is >= a NaN; a place that
      // is a NaN lies in bin 0)
      const float low = c.first > 0 ? (float)c.first : -1.f, high = c.last < FS_BINS - 1 ? (float)(c.last + 1) : __int_as_float(0x7fc00000);
      for (int i = tid; i < groups; i += FS_THREADS) {
        const float4 v = group_of(i);
        const float x[4] = {v.x, v.y, v.z, v.w};
        double w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = place_of(x[e]);
          const bool ahead = p < low || (c.first > 0 && !(p >= 0.f));
          if (x[e] > -INFINITY && !ahead && !(p >= high)) take(x[e], id_of(i, e));
          w[e] = c.want_front && ahead ? 1.0 : 0.0;
        }
        if (c.want_front && w[0] + w[1] + w[2] + w[3] > 0.0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) front += w[e] > 0.0 ? weight(x[e]) : 0ull;
        }
        if (c.want_m) {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = weight.plain(x[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) m_sum += w[e] >= m_border ? weight.whole(w[e]) : 0ull;
        }
      }
    } else {
      const bool by_order = c.what == FS_RADIX || c.what == FS_FETCH_ORDER;
      for (int i = tid; i < groups; i += FS_THREADS) {
        const float4 v = group_of(i);
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const float l = e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
          if (!(l > -INFINITY)) continue;
          bool in, ahead;
          int at;
          if (by_order) {
            const u64 order = fs_order(l, id_of(i, e));
            in = order >= c.low && order <= c.high;
            ahead = order > c.high;
            at = (int)((c.high - order) >> c.shift);
          } else {
            const float x = place_of(l);
            const int b = bin_of(x);
            in = b >= c.first && b <= c.last;
            ahead = b < c.first;
            at = min(FS_BINS - 1, (int)((x - (float)c.first) * c.fine_scale));
            if (in && !cut) {
              ahead = at < c.fine;
              in = at == c.fine;
            }
          }
          if (in && cut) {
            const u64 w = weight(l);
            atomicAdd(&sh.count[at], 1u);
            const unsigned low = (unsigned)w, old = atomicAdd(&low_word[at], low);
            const unsigned high = (unsigned)(w >> 32) + (old + low < old);
            if (high) atomicAdd(&high_word[at], high);
          } else if (in) {
            take(l, id_of(i, e));
          }
          if (ahead) front += weight(l);
          if (c.want_m) {
            const double w = weight.plain(l);
            if (w >= m_border) m_sum += weight.whole(w);
          }
        }
      }
    }
    if (c.want_front) front = block.sum(front);
    if (c.want_m) m_sum = block.sum(m_sum);
    if (tid == 0) tell(front, m_sum);
    if (!cut && rank != 0) {
      __syncthreads();
      const unsigned mine = min(sh.mine, (unsigned)FS_LIST);
      if (mine) {                                  // the same for the block
        const u64 base = block.from(tid == 0, tid == 0 ? fs_add32(&sh.listed, 0, mine) : 0u);
        for (unsigned i = tid; i < mine; i += FS_THREADS)
          if (base + i < FS_LIST) fs_store64(&sh.list[base + i], 0, sh.list[i]);
      }
    }
  };
  if (rank != 0) {
    while (true) {
      fs_sync();                                 // a command is there
      const FsCommand c = sh.command;
      serve(c);
      fs_sync();                                 // it has been carried out
      if (c.is_last) return;
    }
  }

  // ---- 3. the first block decides ----
  auto ask = [&](const FsCommand& c) {
    __syncthreads();
    if (warp == 0) {
      const uint4* words = reinterpret_cast<const uint4*>(&c);
      if (lane < (int)size)
        for (int i = 0; i < (int)(sizeof(FsCommand) / 16); ++i) fs_store128(reinterpret_cast<uint4*>(&sh.command) + i, lane, words[i]);
      if (lane == 0) sh.listed = 0;
    }
    fs_sync();
    serve(c);
    fs_sync();
  };
  auto total_of = [&](int which) {
    u64 v = 0;
    for (unsigned r = 0; r < size; ++r) v += which ? sh.sums[r].y : sh.sums[r].x;
    return v;
  };
  // every bin's count over the cluster, and running counts; bounds on running sums, in units
  unsigned count_of[FS_EACH], count_to[FS_EACH];
  double least_to[FS_EACH], most_to[FS_EACH];
  auto counts = [&]() {
    uint4 v[FS_MAX_CLUSTER];
#pragma unroll
    for (int r = 0; r < FS_MAX_CLUSTER; ++r)
      v[r] = r < (int)size ? fs_load128(&sh.count[tid * FS_EACH], r) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) count_of[i] = 0;
#pragma unroll
    for (int r = 0; r < FS_MAX_CLUSTER; ++r) { count_of[0] += v[r].x; count_of[1] += v[r].y; count_of[2] += v[r].z; count_of[3] += v[r].w; }
  };
  counts();
  const u64 all_sum = by_k ? 0 : total_of(0), m_sum0 = by_k || !by_m ? 0 : total_of(1);
  // An edge's weight in units from the single-precision exponential, widened by 2^-14 of itself (its own error, and what a place
  // is rounded by, are below 2^-16 at the exponents that count); the last bin has no lower edge, nor has any where all
  // candidates are equal or almost.
  const float nats = bin_scale > 0.f ? 1.f / bin_scale : 0.f, step = (float)(nats * rate);
  auto edge = [&](int b) { return b == 0 ? 1.f : exp2f(-(float)b * step); };
  {
    unsigned n_to = 0;
    double least = 0, most = 0;
    float high = edge(tid * FS_EACH);
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) {
      const int b = tid * FS_EACH + i;
      const float low = b == FS_BINS - 1 || !(step > 0.f) ? 0.f : edge(b + 1);
      n_to += count_of[i];
      most += count_of[i] * (fmin((double)high * (1 + 1.0 / 16384), 1.0) * weight.unit + 1);
      least += count_of[i] * fmax((double)low * (1 - 1.0 / 16384) * weight.unit - 1, 0.0);
      count_to[i] = n_to;
      least_to[i] = least;
      most_to[i] = most;
      high = step > 0.f ? low : 1.f;
    }
    block.before(n_to, least, most);
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) { count_to[i] += n_to; least_to[i] += least; most_to[i] += most; }
  }
  // the first of all places (a thread has four) whose test holds; FS_BINS if none does
  auto first_of = [&](auto holds) {
    unsigned at = FS_BINS;
#pragma unroll
    for (int i = FS_EACH - 1; i >= 0; --i)
      if (holds(i)) at = tid * FS_EACH + i;
    return (int)block.min(at);
  };
  // a number that the threads have four of, at a place
  auto at_place = [&](const auto& v, int b) {
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i)
      if ((b & (FS_EACH - 1)) == i) mine = (u64)v[i];
    return block.from(tid == b / FS_EACH, mine);
  };
  // The list, sorted, with its weights' running sums (from `front` on).
  u64 sum_to[FS_EACH], order_at[FS_EACH];
  int in_list = 0;
  auto sorted = [&](u64 front) {
    in_list = min((int)sh.listed, FS_LIST);
    int padded = 128;
    while (padded < in_list) padded <<= 1;
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) order_at[i] = tid * FS_EACH + i < in_list ? sh.list[tid * FS_EACH + i] : 0;
    fs_sort(order_at, sh.list, padded);
    u64 mine = 0;
    if (warp * 32 * FS_EACH < in_list) {
#pragma unroll
      for (int i = 0; i < FS_EACH; ++i) {
        if (tid * FS_EACH + i < in_list) mine += weight(fs_value((unsigned)(order_at[i] >> 32)));
        sum_to[i] = mine;
      }
    } else {
#pragma unroll
      for (int i = 0; i < FS_EACH; ++i) sum_to[i] = 0;
    }
    unsigned none = 0, also_none = 0;
    block.before(mine, none, also_none);
#pragma unroll
    for (int i = 0; i < FS_EACH; ++i) sum_to[i] += mine + front;
  };
  auto in_the_list = [&](int i) { return tid * FS_EACH + i < in_list; };
  auto id_at = [&](int at) { return (int)~(unsigned)at_place(order_at, at); };

  // The border of `goal`: makes the list hold the candidates around it, and returns the first place in the list that reaches
  // it: the goal-th candidate (by_count), or the first whose running sum is > goal (strict) or >= goal.
  auto border = [&](bool by_count, double goal, bool strict, bool want_m) {
    auto reached = [&](double sum) { return strict ? sum > goal : sum >= goal; };
    int first, last;
    if (by_count) {
      first = last = first_of([&](int i) { return (double)count_to[i] >= goal; });
    } else {
      first = first_of([&](int i) { return count_of[i] > 0 && most_to[i] * (1 + 1e-9) >= goal; });
      last = min(FS_BINS - 1, first_of([&](int i) { return least_to[i] * (1 - 1e-9) > goal; }));
      first = min(first, last);
    }
    unsigned passed = first > 0 ? (unsigned)at_place(count_to, first - 1) : 0;      // candidates in front of the list
    const unsigned inside = (unsigned)at_place(count_to, last) - passed;
    FsCommand c{};
    c.what = FS_FETCH;
    c.first = first;
    c.last = last;
    c.want_front = 1;
    if (inside > FS_LIST) {
      // cut finer: by the place below the largest, then by the order itself
      unsigned kept_count[FS_EACH], kept_to[FS_EACH];
#pragma unroll
      for (int i = 0; i < FS_EACH; ++i) { kept_count[i] = count_of[i]; kept_to[i] = count_to[i]; }
      c.what = FS_FINE;
      c.fine_scale = 2047.96875f / (float)(last - first + 1);
      u64 low = (u64)fs_key(all.min) << 32, high = (u64)fs_key(all.max) << 32 | 0xffffffffu;
      while (true) {
        if (c.what == FS_RADIX) {
          c.low = low;
          c.high = high;
          c.shift = 0;
          while ((high - low) >> c.shift >= FS_BINS) ++c.shift;
        }
        ask(c);
        u64 before = total_of(0), sum = 0, to[FS_EACH];
        counts();
        for (unsigned r = 0; r < size; ++r) {
          const uint4 a = fs_load128(reinterpret_cast<unsigned*>(sh.list) + tid * FS_EACH, r);
          const uint4 b = fs_load128(reinterpret_cast<unsigned*>(sh.list) + FS_BINS + tid * FS_EACH, r);
          const u64 w[FS_EACH] = {a.x + ((u64)b.x << 32), a.y + ((u64)b.y << 32), a.z + ((u64)b.z << 32), a.w + ((u64)b.w << 32)};
#pragma unroll
          for (int i = 0; i < FS_EACH; ++i) to[i] = (r ? to[i] : 0) + w[i];
        }
        unsigned n_to = 0, none = 0;
#pragma unroll
        for (int i = 0; i < FS_EACH; ++i) {
          n_to += count_of[i];
          count_to[i] = n_to;
          sum += to[i];
          to[i] = sum;
        }
        block.before(n_to, sum, none);
#pragma unroll
        for (int i = 0; i < FS_EACH; ++i) { count_to[i] += n_to; to[i] += sum + before; }
        const unsigned in_front = passed;
        const int at = min(FS_BINS - 1, first_of([&](int i) {
          return count_of[i] > 0 && (by_count ? (double)(in_front + count_to[i]) >= goal : reached((double)to[i]));
        }));
        const unsigned here = (unsigned)at_place(count_of, at), in_bins = at > 0 ? (unsigned)at_place(count_to, at - 1) : 0;
        if (c.what == FS_FINE) {
          if (here <= FS_LIST) {
            c.what = FS_FETCH_FINE;
            c.fine = at;
            passed += in_bins;
            break;
          }
          c.what = FS_RADIX;                        // from the whole order on
          passed = 0;
        } else {
          const u64 span = (1ull << c.shift) - 1;
          high -= (u64)at << c.shift;
          low = high - low > span ? high - span : low;
          passed += in_bins;
          if (here <= FS_LIST) {
            c.what = FS_FETCH_ORDER;
            c.low = low;
            c.high = high;
            break;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < FS_EACH; ++i) { count_of[i] = kept_count[i]; count_to[i] = kept_to[i]; }
    }
    c.want_m = want_m;
    c.is_last = strict;                             // the draw is the last border
    ask(c);
    sorted(total_of(0));
    const unsigned in_front = passed;
    const int at = first_of([&](int i) {
      return in_the_list(i) && (by_count ? (double)(in_front + tid * FS_EACH + i + 1) >= goal : reached((double)sum_to[i]));
    });
    return max(0, min(at, in_list - 1));
  };

  const double u = u_asked >= 0.f ? fmin((double)u_asked, 1.0 - 1.0 / 16777216) : 0.0;
  int chosen;
  const unsigned candidates = (unsigned)at_place(count_to, FS_BINS - 1);
  const bool k_cuts = by_k && (unsigned)k_asked < candidates;
  // the last bin that can hold a kept candidate: top-k's, the nucleus' (where its sum is known), min-p's (where top-k and top-p do
  // not need what lies behind it), the last one; and whether all up to it fit the list
  const unsigned k_goal = k_cuts ? (unsigned)k_asked : candidates;
  const double p_goal = p_share * (double)all_sum;
  const int end = first_of([&](int i) {
    return count_to[i] >= k_goal || (by_p && !by_k && least_to[i] >= p_goal) ||
           (by_m && !(by_k && by_p) && (double)edge(tid * FS_EACH + i + 1) * (1 + 1.0 / 16384) < m_border);
  });
  if (at_place(count_to, end) <= FS_LIST) {
    FsCommand c{};
    c.what = FS_FETCH;
    c.last = end;
    c.is_last = 1;
    ask(c);
    sorted(0);
    int kept = in_list;
    if (k_cuts) kept = min(kept, k_asked);
    if (by_p) {
      const double goal = p_share * (double)(by_k ? at_place(sum_to, kept - 1) : all_sum);
      kept = min(kept, first_of([&](int i) { return in_the_list(i) && (double)sum_to[i] >= goal; }) + 1);
    }
    if (by_m) {
      const int below = first_of([&](int i) { return in_the_list(i) && weight.plain(fs_value((unsigned)(order_at[i] >> 32))) < m_border; });
      kept = max(1, min(kept, below));
    }
    const double goal = u * (double)at_place(sum_to, kept - 1);
    const int at = first_of([&](int i) { return in_the_list(i) && (double)sum_to[i] > goal; });
    chosen = id_at(min(at, kept - 1));
  } else {
    u64 kept = all_sum, m_kept = m_sum0;
    if (by_k) {
      // the sum of the first k (of all where there are fewer)
      const int at = border(true, (double)k_goal, false, by_m);
      kept = at_place(sum_to, at);
      if (by_m) m_kept = total_of(1);
    }
    if (by_p) {
      const int at = border(false, p_share * (double)kept, false, false);
      const u64 cut = at_place(sum_to, at);
      kept = min(kept, cut);
    }
    if (by_m) kept = min(kept, m_kept);
    chosen = id_at(border(false, u * (double)kept, true, false));
  }
  if (tid == 0) out[row] = chosen;
}

// Blocks a cluster: a row's slices stay in shared memory, two blocks a multiprocessor, up to 8 * 21,000 logits; few rows
// want many short slices, each a chain of passes.
static int fs_cluster(int vocab) { return vocab > 24576 ? 8 : vocab > 8192 ? 4 : vocab > 3000 ? 2 : 1; }

// Draws one id a row of `logits` [n_rows][vocab].  `top_k` (0 or less: off), `top_p` (1 or more: off) and `min_p` (0: off) may be
// null; `uniform` holds numbers from [0, 1).
TOKB200_API int tokb200_sample_filtered(const float* logits, int n_rows, int vocab, const float* temperature, const int* top_k,
                                        const float* top_p, const float* min_p, const float* uniform, int* out,
                                        cudaStream_t stream) {
  if (n_rows <= 0) return TOKB200_OK;
  if (vocab <= 0 || n_rows > (1 << 27)) return TOKB200_BAD_SIZE;
  const int cluster = fs_cluster(vocab);
  const int slice = (vocab + cluster - 1) / cluster;
  constexpr size_t kMost = 200 * 1024;               // of a block's shared memory
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
  static const int overlap = [] {
    const char* v = getenv("TOKB200_PDL");
    return (v && v[0] == '0') ? 0 : 1;
  }();
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = overlap;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = (unsigned)cluster;
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&config, sample_filtered_kernel, logits, vocab, slice, (int)resident, unit_bits,
                                             temperature, top_k, top_p, min_p, uniform, out);
  return err == cudaSuccess ? TOKB200_OK : (int)err;
}
