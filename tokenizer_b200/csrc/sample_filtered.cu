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
#define FS_BINS 2048
#define FS_LIST 2048
#define FS_MAX_CLUSTER 8
#define FS_BINS_EACH (FS_BINS / FS_THREADS)

typedef unsigned long long u64;

enum : int { FS_DONE = 0, FS_FETCH = 1, FS_FINE = 2, FS_FETCH_FINE = 3, FS_RADIX = 4, FS_FETCH_ORDER = 5 };

// what the first block asks of the cluster: candidates of bins first..last (cut into finer bins with `fine_scale`, of which
// fine_first..fine_last), or those whose place in the order lies in low..high (cut by `shift`)
struct FsCommand {
  int what, first, last, fine_first, fine_last, shift;
  float fine_scale;
  u64 low, high;
};

struct FsStats { float max, min; int id, odd; };       // of a block's slice; odd: it holds a NaN or +infinity

__device__ __forceinline__ unsigned fs_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned fs_size() { unsigned r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void fs_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ unsigned fs_peer(const void* local, unsigned rank) {
  unsigned theirs;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"((unsigned)__cvta_generic_to_shared(local)), "r"(rank));
  return theirs;
}
__device__ __forceinline__ unsigned fs_load32(const void* local, unsigned rank) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(fs_peer(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 fs_load64(const void* local, unsigned rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(fs_peer(local, rank)) : "memory");
  return v;
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

__device__ __forceinline__ u64 fs_warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// block-wide sum; every thread has it
__device__ __forceinline__ u64 fs_block_sum(u64 v, u64* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = fs_warp_sum(v);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  u64 all = 0;
#pragma unroll
  for (int w = 0; w < FS_THREADS / 32; ++w) all += scratch[w];
  return all;
}
// sums of the threads in front of this one
template <typename T>
__device__ __forceinline__ T fs_before(T v, T* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T below = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += below;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  T front = 0;
#pragma unroll
  for (int w = 0; w < FS_THREADS / 32; ++w)
    if (w < warp) front += scratch[w];
  return front + sum - v;
}

struct FsShared {
  u64 list[FS_LIST];                 // candidates; the sums of finer bins take the same place, low and high words
  unsigned count[FS_BINS];
  u64 sums[3];                       // of this block: all weights (or those in front), those above min-p's border, their number
  u64 scratch[FS_THREADS / 32];
  double table[64];
  FsCommand command;
  FsStats stats;
  FsStats of_warps[FS_THREADS / 32];
  unsigned listed;
  int found;
};

// The first place (of FS_BINS_EACH a thread, in order) whose test holds, the number of places if none does.
__device__ __forceinline__ int fs_first(const bool (&test)[FS_BINS_EACH], int* found) {
  __syncthreads();
  if (threadIdx.x == 0) *found = FS_BINS;
  __syncthreads();
#pragma unroll
  for (int i = FS_BINS_EACH - 1; i >= 0; --i)
    if (test[i]) atomicMin(found, (int)threadIdx.x * FS_BINS_EACH + i);
  __syncthreads();
  return *found;
}

__device__ __forceinline__ void fs_sort(u64* list, int n) {      // descending; n a power of two
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += FS_THREADS) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
      }
    }
  __syncthreads();
}

__global__ void __launch_bounds__(FS_THREADS, 2)
sample_filtered_kernel(const float* __restrict__ logits, int vocab, int slice, int resident, int unit_bits,
                       const float* __restrict__ temperature, const int* __restrict__ top_k, const float* __restrict__ top_p,
                       const float* __restrict__ min_p, const float* __restrict__ uniform, int* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char fs_raw[];
  FsShared& sh = *reinterpret_cast<FsShared*>(fs_raw);
  float* held = reinterpret_cast<float*>(fs_raw + sizeof(FsShared));
  const int tid = threadIdx.x;
  const unsigned rank = fs_rank(), size = fs_size();
  const int row = blockIdx.x / size;
  const int begin = min((long long)vocab, (long long)rank * slice), n = min(slice, vocab - begin);
  for (int i = tid; i < FS_BINS; i += FS_THREADS) sh.count[i] = 0;
  if (tid < 64) sh.table[tid] = exp2(tid / 64.0);
  if (tid == 0) sh.listed = 0;
  pdl_wait();
  pdl_launch();
  const float* global = logits + (size_t)row * vocab + begin;
  const float temp = temperature[row];
  const bool greedy = !(temp > 0.f);
  const int k_asked = top_k ? top_k[row] : 0;
  const float p_asked = top_p ? top_p[row] : 1.f, m_asked = min_p ? min_p[row] : 0.f;

  // ---- 1. the slice into shared memory; its largest, smallest finite, and odd values ----
  FsStats mine{-INFINITY, INFINITY, -1, 0};
  constexpr int kAhead = 8;
  for (int i0 = tid; i0 < n; i0 += kAhead * FS_THREADS) {
    float v[kAhead];
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int i = i0 + e * FS_THREADS;
      v[e] = i < n ? global[i] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < kAhead; ++e) {
      const int i = i0 + e * FS_THREADS;
      if (i < n && resident) held[i] = v[e];
      if (v[e] > mine.max) { mine.max = v[e]; mine.id = begin + i; }
      if (v[e] > -INFINITY) mine.min = fminf(mine.min, v[e]);
      if (!(v[e] < INFINITY)) mine.odd = 1;
    }
  }
  auto join = [](FsStats& a, const FsStats& b) {
    if (b.id >= 0 && (a.id < 0 || b.max > a.max || (b.max == a.max && b.id < a.id))) { a.max = b.max; a.id = b.id; }
    a.min = fminf(a.min, b.min);
    a.odd |= b.odd;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    join(mine, FsStats{__shfl_xor_sync(0xffffffffu, mine.max, o), __shfl_xor_sync(0xffffffffu, mine.min, o),
                       __shfl_xor_sync(0xffffffffu, mine.id, o), __shfl_xor_sync(0xffffffffu, mine.odd, o)});
  if ((tid & 31) == 0) sh.of_warps[tid >> 5] = mine;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < FS_THREADS / 32; ++w) join(mine, sh.of_warps[w]);
    sh.stats = mine;
  }
  fs_sync();
  FsStats all{-INFINITY, INFINITY, -1, 0};
  for (unsigned r = 0; r < size; ++r)
    join(all, FsStats{__uint_as_float(fs_load32(&sh.stats.max, r)), __uint_as_float(fs_load32(&sh.stats.min, r)),
                      (int)fs_load32(&sh.stats.id, r), (int)fs_load32(&sh.stats.odd, r)});
  // greedy rows; rows whose weights have no finite sum; rows without a candidate
  if (greedy || all.odd || all.id < 0) {
    if (rank == 0 && tid == 0) out[row] = all.id < 0 ? 0 : all.id;
    fs_sync();                                   // nobody leaves while its values may still be read
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
  const float* vals = resident ? held : global;
  {
    u64 sum = 0, m_sum = 0, m_count = 0;
    for (int i = tid; i < n; i += FS_THREADS) {
      const float l = vals[i];
      if (!(l > -INFINITY)) continue;
      atomicAdd(&sh.count[bin_of(place_of(l))], 1u);
      if (!by_k) {
        const double w = weight.plain(l);
        const u64 whole = weight.whole(w);
        sum += whole;
        if (by_m && w >= m_border) { m_sum += whole; ++m_count; }
      }
    }
    if (!by_k) {
      sum = fs_block_sum(sum, sh.scratch);
      if (by_m) { m_sum = fs_block_sum(m_sum, sh.scratch); m_count = fs_block_sum(m_count, sh.scratch); }
    }
    if (tid == 0) { sh.sums[0] = sum; sh.sums[1] = m_sum; sh.sums[2] = m_count; }
  }
  fs_sync();

  // ---- the others do what the first block asks ----
  auto serve = [&](const FsCommand& c) {
    const bool by_order = c.what == FS_RADIX || c.what == FS_FETCH_ORDER;
    const bool cut = c.what == FS_FINE || c.what == FS_RADIX;
    u64 front = 0, m_sum = 0;
    unsigned* low_word = reinterpret_cast<unsigned*>(sh.list);
    unsigned* high_word = low_word + FS_BINS;
    if (cut) {
      // the first block's list of bins is in its threads' registers by now, and so are the others' counts in its own
      for (int i = tid; i < FS_BINS; i += FS_THREADS) { sh.count[i] = 0; low_word[i] = 0; high_word[i] = 0; }
      __syncthreads();
    }
    for (int i = tid; i < n; i += FS_THREADS) {
      const float l = vals[i];
      if (!(l > -INFINITY)) continue;
      bool in;
      int at = 0;
      bool ahead;
      const u64 order = fs_order(l, begin + i);
      if (by_order) {
        in = order >= c.low && order <= c.high;
        ahead = order > c.high;
        at = (int)((c.high - order) >> c.shift);
      } else {
        const float x = place_of(l);
        const int b = bin_of(x);
        in = b >= c.first && b <= c.last;
        ahead = b < c.first;
        if (c.what != FS_FETCH) {
          at = min(FS_BINS - 1, (int)((x - (float)c.first) * c.fine_scale));
          if (in && c.what == FS_FETCH_FINE) {
            ahead = at < c.fine_first;
            in = at >= c.fine_first && at <= c.fine_last;
          }
        }
      }
      if (cut && in) {
        const u64 w = weight(l);
        atomicAdd(&sh.count[at], 1u);
        const unsigned low = (unsigned)w, old = atomicAdd(&low_word[at], low);
        const unsigned high = (unsigned)(w >> 32) + (old + low < old);
        if (high) atomicAdd(&high_word[at], high);
      } else if (in) {
        const unsigned to = fs_add32(&sh.listed, 0, 1u);
        if (to < FS_LIST) fs_store64(&sh.list[to], 0, order);
      }
      if (ahead) front += weight(l);
      if (by_m && by_k && !cut && weight.plain(l) >= m_border) m_sum += weight(l);
    }
    front = fs_block_sum(front, sh.scratch);
    if (by_m && by_k && !cut) m_sum = fs_block_sum(m_sum, sh.scratch);
    if (tid == 0) { sh.sums[0] = front; sh.sums[1] = m_sum; }
  };
  if (rank != 0) {
    while (true) {
      fs_sync();                                 // a command is there
      FsCommand c;
      c.what = (int)fs_load32(&sh.command.what, 0);
      c.first = (int)fs_load32(&sh.command.first, 0);
      c.last = (int)fs_load32(&sh.command.last, 0);
      c.fine_first = (int)fs_load32(&sh.command.fine_first, 0);
      c.fine_last = (int)fs_load32(&sh.command.fine_last, 0);
      c.shift = (int)fs_load32(&sh.command.shift, 0);
      c.fine_scale = __uint_as_float(fs_load32(&sh.command.fine_scale, 0));
      c.low = fs_load64(&sh.command.low, 0);
      c.high = fs_load64(&sh.command.high, 0);
      if (c.what == FS_DONE) break;
      serve(c);
      fs_sync();                                 // it has been carried out
    }
    fs_sync();
    return;
  }

  // ---- 3. the first block decides ----
  auto ask = [&](const FsCommand& c) {
    __syncthreads();
    if (tid == 0) { sh.command = c; sh.listed = 0; }
    fs_sync();
    if (c.what != FS_DONE) {
      serve(c);
      fs_sync();
    }
  };
  auto total_of = [&](int which) {
    u64 v = 0;
    for (unsigned r = 0; r < size; ++r) v += fs_load64(&sh.sums[which], r);
    return v;
  };
  // every bin's count over the cluster, and running counts; bounds on running sums, in units
  unsigned count_of[FS_BINS_EACH], count_to[FS_BINS_EACH];
  double least_to[FS_BINS_EACH], most_to[FS_BINS_EACH];
  auto counts = [&]() {
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) count_of[i] = 0;
    for (unsigned r = 0; r < size; ++r)
#pragma unroll
      for (int i = 0; i < FS_BINS_EACH; ++i) count_of[i] += fs_load32(&sh.count[tid * FS_BINS_EACH + i], r);
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) { mine += count_of[i]; count_to[i] = mine; }
    const unsigned front = fs_before<unsigned>(mine, reinterpret_cast<unsigned*>(sh.scratch));
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) count_to[i] += front;
  };
  counts();
  const u64 all_sum = by_k ? 0 : total_of(0), m_sum0 = by_k || !by_m ? 0 : total_of(1);
  {
    double least = 0, most = 0;
    const double nats = bin_scale > 0.f ? 1.0 / (double)bin_scale : 0.0;
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) {
      const int b = tid * FS_BINS_EACH + i;
      // a place is rounded twice; the last bin has no lower edge, nor has any where all candidates are equal or almost
      const double high = exp2(-b * nats * (1 - 4e-7) * rate), low = b == FS_BINS - 1 || nats == 0.0 ? 0.0 : exp2(-(b + 1) * nats * (1 + 4e-7) * rate);
      most += count_of[i] * (fmin(high, 1.0) * weight.unit * (1 + 1e-9) + 1);
      least += count_of[i] * fmax(low * weight.unit * (1 - 1e-9) - 1, 0.0);
      least_to[i] = least;
      most_to[i] = most;
    }
    const double least_front = fs_before<double>(least, reinterpret_cast<double*>(sh.scratch));
    const double most_front = fs_before<double>(most, reinterpret_cast<double*>(sh.scratch));
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) { least_to[i] += least_front; most_to[i] += most_front; }
  }
  bool test[FS_BINS_EACH];
  auto first_bin = [&](auto holds) {
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) test[i] = holds(i);
    return fs_first(test, &sh.found);
  };
  // a thread's register, from the thread that has bin b
  auto of_bin = [&](const unsigned (&v)[FS_BINS_EACH], int b) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i)
      if (tid * FS_BINS_EACH + i == b) sh.found = (int)v[i];
    __syncthreads();
    return (unsigned)sh.found;
  };
  // The list, sorted, its weights and running sums (from `front` on) four to a thread.
  u64 sum_to[FS_BINS_EACH], order_at[FS_BINS_EACH];
  int in_list = 0;
  auto sorted = [&](u64 front) {
    in_list = min((int)sh.listed, FS_LIST);
    int padded = 2;
    while (padded < in_list) padded <<= 1;
    for (int i = in_list + tid; i < padded; i += FS_THREADS) sh.list[i] = 0;
    fs_sort(sh.list, padded);
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) {
      const int at = tid * FS_BINS_EACH + i;
      order_at[i] = at < in_list ? sh.list[at] : 0;
      if (at < in_list) mine += weight(fs_value((unsigned)(order_at[i] >> 32)));
      sum_to[i] = mine;
    }
    const u64 before = fs_before<u64>(mine, sh.scratch);
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i) sum_to[i] += before + front;
  };
  auto in_the_list = [&](int i) { return tid * FS_BINS_EACH + i < in_list; };
  auto sum_at = [&](int at) -> u64 {               // running sum at a place of the list
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FS_BINS_EACH; ++i)
      if (tid * FS_BINS_EACH + i == at) sh.scratch[0] = sum_to[i];
    __syncthreads();
    const u64 v = sh.scratch[0];
    __syncthreads();
    return v;
  };
  auto id_at = [&](int at) { return (int)~(unsigned)sh.list[at]; };

  // The border of `goal`: makes the list hold the candidates around it, and returns the first place in the list that
  // reaches it.  by_count: the goal-th candidate; else the first whose running sum is > goal (strict) or >= goal.
  auto border = [&](bool by_count, double goal, bool strict) {
    auto reached = [&](double sum) { return strict ? sum > goal : sum >= goal; };
    int first, last;
    unsigned passed;                                // candidates in front of the list
    if (by_count) {
      first = last = first_bin([&](int i) { return (double)count_to[i] >= goal; });
    } else {
      first = first_bin([&](int i) { return count_of[i] > 0 && most_to[i] >= goal * (1 - 1e-9); });
      last = first_bin([&](int i) { return least_to[i] * (1 - 1e-9) > goal; });
      if (last >= FS_BINS) last = FS_BINS - 1;
      if (first > last) first = last;
    }
    passed = first > 0 ? of_bin(count_to, first - 1) : 0;
    const unsigned inside = of_bin(count_to, last) - passed;
    FsCommand c{FS_FETCH, first, last, 0, 0, 0, 0.f, 0, 0};
    if (inside > FS_LIST) {
      // cut finer: by the place below the largest, then by the order itself
      unsigned kept_count[FS_BINS_EACH], kept_to[FS_BINS_EACH];
      double kept_least[FS_BINS_EACH], kept_most[FS_BINS_EACH];
#pragma unroll
      for (int i = 0; i < FS_BINS_EACH; ++i) {
        kept_count[i] = count_of[i]; kept_to[i] = count_to[i]; kept_least[i] = least_to[i]; kept_most[i] = most_to[i];
      }
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
        const u64 front = total_of(0);
        counts();
        unsigned* low_word = reinterpret_cast<unsigned*>(sh.list);
        unsigned* high_word = low_word + FS_BINS;
        u64 mine = 0, to[FS_BINS_EACH];
#pragma unroll
        for (int i = 0; i < FS_BINS_EACH; ++i) {
          for (unsigned r = 0; r < size; ++r)
            mine += fs_load32(&low_word[tid * FS_BINS_EACH + i], r) + ((u64)fs_load32(&high_word[tid * FS_BINS_EACH + i], r) << 32);
          to[i] = mine;
        }
        const u64 before = fs_before<u64>(mine, sh.scratch) + front;
        // candidates in front of what was cut: those of the bins in front, or of what the order's cuts left behind
        const unsigned cut_front = passed;
        const int at = min(FS_BINS - 1, first_bin([&](int i) {
          return count_of[i] > 0 && (by_count ? (double)(cut_front + count_to[i]) >= goal : reached((double)(before + to[i])));
        }));
        const unsigned here = of_bin(count_of, at), in_front = at > 0 ? of_bin(count_to, at - 1) : 0;
        if (c.what == FS_FINE) {
          if (here <= FS_LIST) {
            c.what = FS_FETCH_FINE;
            c.fine_first = c.fine_last = at;
            passed += in_front;
            break;
          }
          c.what = FS_RADIX;                        // from the whole order on
          passed = 0;
        } else {
          const u64 top = high - ((u64)at << c.shift);
          const u64 span = (1ull << c.shift) - 1;
          low = top - low > span ? top - span : low;
          high = top;
          passed += in_front;
          if (here <= FS_LIST) {
            c.what = FS_FETCH_ORDER;
            c.low = low;
            c.high = high;
            break;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < FS_BINS_EACH; ++i) {
        count_of[i] = kept_count[i]; count_to[i] = kept_to[i]; least_to[i] = kept_least[i]; most_to[i] = kept_most[i];
      }
    }
    ask(c);
    sorted(total_of(0));
    const unsigned in_front = passed;
    int at = first_bin([&](int i) {
      return in_the_list(i) && (by_count ? (double)(in_front + tid * FS_BINS_EACH + i + 1) >= goal : reached((double)sum_to[i]));
    });
    return max(0, min(at, in_list - 1));
  };

  const float u_row = uniform[row];
  const double u = u_row >= 0.f ? fmin((double)u_row, 1.0 - 1.0 / 16777216) : 0.0;
  int chosen;
  // the last bin that can hold a kept candidate, and whether all up to it fit the list
  const unsigned candidates = of_bin(count_to, FS_BINS - 1);
  const bool k_cuts = by_k && (unsigned)k_asked < candidates;
  int end = first_bin([&](int i) { return count_to[i] >= (k_cuts ? (unsigned)k_asked : candidates); });
  if (!by_k && by_p) end = min(end, first_bin([&](int i) { return least_to[i] >= p_share * (double)all_sum; }));
  if (by_m) {
    const double nats = bin_scale > 0.f ? 1.0 / (double)bin_scale : 0.0;
    // candidates behind this bin have weights below the border
    const int m_end = first_bin([&](int i) { return exp2(-(tid * FS_BINS_EACH + i + 1) * nats * (1 - 4e-7) * rate) < m_border * (1 - 1e-9); });
    if (!by_k || !by_p) end = min(end, min(m_end, FS_BINS - 1));
  }
  if (of_bin(count_to, end) <= FS_LIST) {
    ask(FsCommand{FS_FETCH, 0, end, 0, 0, 0, 0.f, 0, 0});
    sorted(0);
    int kept = in_list;
    if (k_cuts) kept = min(kept, k_asked);
    if (by_p) {
      const double goal = p_share * (double)(by_k ? sum_at(kept - 1) : all_sum);
      kept = min(kept, first_bin([&](int i) { return in_the_list(i) && (double)sum_to[i] >= goal; }) + 1);
    }
    if (by_m) {
      const int below = first_bin([&](int i) { return in_the_list(i) && weight.plain(fs_value((unsigned)(order_at[i] >> 32))) < m_border; });
      kept = max(1, min(kept, below));
    }
    const double goal = u * (double)sum_at(kept - 1);
    const int at = first_bin([&](int i) { return in_the_list(i) && (double)sum_to[i] > goal; });
    chosen = id_at(min(at, kept - 1));
  } else {
    u64 kept = all_sum, m_kept = m_sum0;
    if (by_k) {
      // the sum of the first k (of all where there are fewer)
      const int at = border(true, (double)(k_cuts ? (unsigned)k_asked : candidates), false);
      kept = sum_at(at);
      if (by_m) m_kept = total_of(1);
    }
    if (by_p) {
      const int at = border(false, p_share * (double)kept, false);
      kept = min(kept, sum_at(at));
    }
    if (by_m) kept = min(kept, m_kept);
    const int at = border(false, u * (double)kept, true);
    chosen = id_at(at);
  }
  __syncthreads();
  if (tid == 0) out[row] = chosen;
  ask(FsCommand{FS_DONE, 0, 0, 0, 0, 0, 0.f, 0, 0});
  fs_sync();
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
  const bool resident = sizeof(FsShared) + (size_t)slice * 4 <= kMost;
  const size_t smem = sizeof(FsShared) + (resident ? (size_t)slice * 4 : 0);
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
