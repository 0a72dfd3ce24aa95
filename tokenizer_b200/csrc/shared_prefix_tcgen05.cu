// Attention of decoding rows whose caches begin with the same pages, on the tensor cores (bfloat16, heads of 64 or 128 lanes,
// pages of a multiple of 8 keys, groups of up to 16 heads).  The definition and what a part of a softmax is are in
// shared_prefix.cu.  Two kernels:
//
// 1. The common keys on tcgen05.  A tile's (member, head) pairs of one key/value head are the 128 rows of a product, two such
//    products (two lanes of work) a block, so that keys and values are read once for up to 256 pairs; a tile with no more
//    than 128 pairs has its key blocks dealt out to the two lanes.  The walk over key blocks, the roles of the warps, the softmax
//    and the place of everything in tensor memory are those of attention_tcgen05.cu; here no key is masked but behind the end,
//    the rows of q are gathered by threads, and what a block leaves is a part: weighted values, maximum and sum in 32 bits.
//    The keys are cut into as many pieces as fill the device once.
// 2. The own keys on mma.sync, and the join.  A cluster of blocks a (row, key/value head): each block walks a piece of the row's
//    own keys, the group's heads as one product (a warp takes 32 keys a turn; the next keys are asked for when the scores are
//    computed, the next values when the weighted sum is); the pieces meet in distributed shared memory, and each block joins
//    every size-th head with the parts of the first kernel.
// Rounding: both kernels round a weight to bfloat16 in front of the second product, half a step (2^-8 of it at most), as the
// framework's other attention on tensor cores does (a second product for what the rounding leaves would double that one's time);
// sums of weights, weighted values and everything that is joined stay in 32 bits.  4 to 64 rows behind 512 to 8,192
// keys are 0.0019 to 0.0023 off 64 bits (relative 2-norm), where the output's own rounding is 0.0017; the same inputs give the same bits.
//
// The first kernel lets the second start at once: what it reads but the parts (rows, tables, q, keys and values) was complete
// before the first kernel began, which starts strictly behind its predecessor.  Its blocks take the multiprocessors that the
// first kernel leaves and those that it has done with, and wait for it only in front of the join.
//
// 64 rows of 28 heads over 4 of 128 lanes, 8,192 common keys and 256 to 1,024 own ones: 36.7 us on the device for 101 MB (2.7 TB/s);
// the common keys' parts are stored at 29.6, the last own keys walked at 27, the join runs from 31.6 to 33.6.  The own keys alone
// take 28.4 us for 82 MB.  16 rows of 12 over 2 behind 4,096: 13.2 us, mostly the two kernels' starts and ends.
#define FA_WAIT_LIMIT (1u << 17)      // polls of up to 20 us each: seconds in all
#ifndef HEAD_DIM
#define HEAD_DIM 64
#endif
static_assert(HEAD_DIM == 64 || HEAD_DIM == 128, "head size");
#define SP_ROWS 128
#define SP_KEYS 128
#define SP_SOFTMAX_WARPS 16             // eight a lane
#define SP_LOADER_WARPS 2
#define SP_THREADS ((SP_SOFTMAX_WARPS + SP_LOADER_WARPS + 1) * 32)
#define SP_BUFFERS (HEAD_DIM == 64 ? 8 : 5)
#define SP_RESCALE_AT 8.0f            // log2 units the maximum may lead its reference by
#define SP_MAX_PIECES 24              // of a tile's keys: with the own ones' at most a lane each in the join
constexpr int kDBlocks = HEAD_DIM / 64;           // 64-lane pieces of the head (128 bytes a row)
constexpr int kSubTile = 128 * 128;               // bytes of a [128 x 64] bfloat16 swizzled tile
constexpr int kTmemCols = 512;
// tensor memory as in attention_tcgen05.cu: scores of the lanes at 0 and 128, accumulators at 256 and 384, probabilities behind
// accumulators of 64 columns or on the first half of the scores
constexpr bool kPOnScores = HEAD_DIM == 128;
constexpr int kPFirst = kPOnScores ? 0 : 256 + HEAD_DIM;
constexpr int kHalfKeys = SP_KEYS / 2;            // of a block, that a softmax thread owns
constexpr int kTileBytes = kDBlocks * kSubTile;
constexpr int kStatBytes = 2 * 2 * SP_ROWS * 4;
constexpr int kBarBytes = (2 * SP_BUFFERS + 7) * 8 + 8;     // the barriers, where tensor memory lies, whether a wait ran out
constexpr int kFaSmem = 2 * kTileBytes + SP_BUFFERS * kTileBytes + kStatBytes + kBarBytes;
static_assert(kFaSmem > 116 * 1024 && kFaSmem <= 227 * 1024, "one block an SM: it takes all of tensor memory");
constexpr int kOutStride = HEAD_DIM * 4 + 16;     // bytes between the rows of a part on their way out through the ring's memory
static_assert(2 * SP_ROWS * kOutStride <= SP_BUFFERS * kTileBytes, "the rows of two lanes fit the ring");

#include "fa_tcgen05.cuh"

__device__ int sp_error_flag = 0;

// keys of a piece when n keys are cut into at most `pieces`: whole blocks
__host__ __device__ __forceinline__ int sp_piece(int n, int pieces) {
  const int len = ((n + pieces - 1) / pieces + SP_KEYS - 1) / SP_KEYS * SP_KEYS;
  return len < SP_KEYS ? SP_KEYS : len;
}

// whether a tile has at most `most` members, all of them in a list of `n_listed`
__device__ __forceinline__ bool sp_tile_fits(const int4& tile, int most, int n_listed) {
  return tile.y <= 0 || (tile.y <= most && tile.x >= 0 && tile.x <= n_listed - tile.y);
}

// the request whose table a tile's keys are read through: its first live member's (-1: it has none)
__device__ __forceinline__ int sp_tile_request(const int4& tile, const int* __restrict__ members, const int* __restrict__ row_req, int n_rows) {
  int req = -1;
  for (int i = 0; i < tile.y && req < 0; ++i) {
    const int row = members[tile.x + i];
    if (row >= n_rows && threadIdx.x == 0) tokb200_report_error(TOKB200_LIB_SHARED_PREFIX_TCGEN05, 3);
    req = row < 0 || row >= n_rows ? -1 : row_req[row];
  }
  return req;
}

// acc_parts: [row][head][pieces][HEAD_DIM]; stat_parts: [row][head][pieces] (maximum in log2 units, sum)
template <bool CAPPED>
__global__ void __launch_bounds__(SP_THREADS, 1)
shared_prefix_tcgen05_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                             const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ v_pool,
                             const int* __restrict__ block_table, int table_stride, const int* __restrict__ row_req,
                             const int* __restrict__ members, int n_listed, const int4* __restrict__ tiles, int n_rows, int nh, int nkv, int page,
                             int run, int pool_rows, int pieces, float scale_log2, float cap_in, float cap_out,
                             float* __restrict__ acc_parts, float2* __restrict__ stat_parts) {
  unsigned char* q_s = fa_raw;                                   // lane 0, lane 1
  unsigned char* ring = q_s + 2 * kTileBytes;
  float* stat_s = reinterpret_cast<float*>(ring + SP_BUFFERS * kTileBytes);   // [lane][half][row]
  unsigned long long* bars = reinterpret_cast<unsigned long long*>(ring + SP_BUFFERS * kTileBytes + kStatBytes);
  unsigned long long* full = bars;                               // [buffers]: a tile is in place
  unsigned long long* empty = full + SP_BUFFERS;                 // [buffers]: commit of its last reader
  unsigned long long* s_full = empty + SP_BUFFERS;               // [2], commit of Q K^T
  unsigned long long* p_ready = s_full + 2;                      // [2], an arrival per softmax warp of the lane
  unsigned long long* pv_done = p_ready + 2;                     // [2], commit of P V
  unsigned long long* q_full = pv_done + 2;                      // an arrival a softmax warp
  unsigned* tmem_slot = reinterpret_cast<unsigned*>(q_full + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int piece = blockIdx.x, kvh = blockIdx.y, group = nh / nkv;
  constexpr int kMmaWarp = SP_SOFTMAX_WARPS + SP_LOADER_WARPS;
  if (warp == SP_SOFTMAX_WARPS && lane < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &map_k : &map_v) : "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < SP_BUFFERS; ++i) {
      fa_mbar_init(&full[i], 1);
      fa_mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      fa_mbar_init(&s_full[i], 1);
      fa_mbar_init(&p_ready[i], SP_SOFTMAX_WARPS / 2);
      fa_mbar_init(&pv_done[i], 1);
    }
    fa_mbar_init(q_full, SP_SOFTMAX_WARPS);
    tmem_slot[1] = 0;                            // no wait has run out
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(fa_smem(tmem_slot)), "r"((unsigned)kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();
  pdl_launch();
  const int4 tile = tiles[blockIdx.z];
  const int lane_members = SP_ROWS / group;            // members a lane
  const bool fits = sp_tile_fits(tile, 2 * lane_members, n_listed);
  if (!fits && threadIdx.x == 0) tokb200_report_error(TOKB200_LIB_SHARED_PREFIX_TCGEN05, 3);
  const int req = fits ? sp_tile_request(tile, members, row_req, n_rows) : -1;
  const bool aligned = (fa_smem(fa_raw) & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) {
    atomicExch(&sp_error_flag, 2);
    tokb200_report_error(TOKB200_LIB_SHARED_PREFIX_TCGEN05, 2);
  }
  const int keys = min(tile.z, table_stride * page), len = sp_piece(keys, pieces);
  const int first = piece * len, end = min(keys, first + len);
  const bool live = aligned && req >= 0 && first < end;
  const int n_blocks = live ? (end - first + SP_KEYS - 1) / SP_KEYS : 0;
  const int n_members = tile.y;
  const bool split = n_members <= lane_members;      // a tile that one lane holds is split along its keys
  auto rows_of = [&](int l) { return group * (split || l == 0 ? min(n_members, lane_members) : n_members - lane_members); };
  auto member_of = [&](int l, int r) { return members[tile.x + (split ? 0 : l * lane_members) + r / group]; };
  auto steps_of = [&](int l) { return split ? (n_blocks + 1 - l) / 2 : n_blocks; };
  auto block_of = [&](int l, int b) { return split ? 2 * b + l : b; };
  // the ring's sequence of tiles: K0 V0 K1 V1 ... side by side, K0 K1 V0 K2 V1 K3 ... split (in the order of their use; a
  // split walk's place for the keys behind the last block stays empty, nothing comes behind it in its buffer)
  auto k_place = [&](int b) { return split ? (b < 2 ? b : 2 * b - 1) : 2 * b; };
  auto v_place = [&](int b) { return split ? 2 * b + 2 : 2 * b + 1; };
  auto of_values = [&](int n) { return split ? n >= 2 && n % 2 == 0 : n % 2 == 1; };
  auto block_at = [&](int n) { return !split ? n / 2 : n < 2 ? n : n % 2 == 0 ? n / 2 - 1 : (n + 1) / 2; };
  const int* table = block_table + (size_t)(live ? req : 0) * table_stride;

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (live && warp >= SP_SOFTMAX_WARPS && warp < kMmaWarp) {
    // ---------------- loaders: the places in turn, a copy a run of keys inside one page ----------------
    const int loader = warp - SP_SOFTMAX_WARPS;
    const int n_places = v_place(n_blocks - 1) + 1, runs = SP_KEYS / run;      // at most 16 runs: a lane each
    // a place's block and whether it is values; this lane's run of keys: its pool row (behind the pool: zeros), and whether
    // some or all of it lies in front of the end
    struct Place { int b, y; bool values, some, all; };
    auto locate = [&](int n) {
      Place at;
      at.values = of_values(n);
      at.b = block_at(n);
      at.y = pool_rows;
      at.some = at.all = false;
      if (n < n_places && at.b < n_blocks && lane < runs) {
        const int key0 = first + at.b * SP_KEYS + lane * run;
        at.some = key0 < end;
        at.all = key0 + run <= end;
        if (at.some) at.y = max(table[key0 / page], 0) * page + key0 % page;
      }
      return at;
    };
    int n = loader;
    Place next = locate(n);
#pragma unroll 1
    for (; n < n_places; n += SP_LOADER_WARPS) {
      const Place at = next;
      next = locate(n + SP_LOADER_WARPS);
      if (at.b >= n_blocks) continue;
      const int buf = n % SP_BUFFERS, use = n / SP_BUFFERS;
      if (use > 0 && !__all_sync(0xffffffffu, fa_mbar_wait(&empty[buf], (use - 1) & 1))) break;
      unsigned char* dst = ring + buf * kTileBytes;
      const unsigned mixed = __ballot_sync(0xffffffffu, at.values && at.some && !at.all);
      if (mixed) {                                     // values that end inside the run: zeros for the others
#pragma unroll 1
        for (unsigned left = mixed; left; left &= left - 1) {
          const int i = __ffs(left) - 1;
          const int row = __shfl_sync(0xffffffffu, at.y, i), key0 = first + at.b * SP_KEYS + i * run;
#pragma unroll 1
          for (int e = lane; e < run * (HEAD_DIM / 8); e += 32) {
            const int t = e / (HEAD_DIM / 8), c = e % (HEAD_DIM / 8);
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (key0 + t < end)
              v = *reinterpret_cast<const uint4*>(v_pool + ((size_t)(row + t) * nkv + kvh) * HEAD_DIM + c * 8);
            *reinterpret_cast<uint4*>(dst + (c / 8) * kSubTile + swz(i * run + t, c % 8)) = v;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      if (lane == 0) fa_expect(&full[buf], (unsigned)(kTileBytes - __popc(mixed) * run * HEAD_DIM * 2));
      __syncwarp();
      if (lane < runs && !(mixed >> lane & 1u)) {
#pragma unroll
        for (int c = 0; c < kDBlocks; ++c)
          fa_tma(dst + c * kSubTile + lane * run * 128, at.values ? &map_v : &map_k, &full[buf], kvh * HEAD_DIM + c * 64, at.y);
      }
      __syncwarp();
    }
    // every copy has landed before the block gives its shared memory back, whatever became of its readers
    const int stop = min(n, n_places);
#pragma unroll 1
    for (int i = loader; i < stop; i += SP_LOADER_WARPS)
      if (i >= stop - SP_BUFFERS && locate(i).b < n_blocks) fa_mbar_wait(&full[i % SP_BUFFERS], (i / SP_BUFFERS) & 1);
  } else if (live && warp == kMmaWarp) {
    // ---------------- products ----------------
    const bool leader = fa_elect();
    constexpr unsigned idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(SP_KEYS >> 3) << 17) |
                                 ((unsigned)(SP_ROWS >> 4) << 24);
    constexpr unsigned idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) /* v is MN-major */ |
                                 ((unsigned)(HEAD_DIM >> 3) << 17) | ((unsigned)(SP_ROWS >> 4) << 24);
    const unsigned q_at = (fa_smem(q_s) & 0x3FFFFu) >> 4, ring_at = (fa_smem(ring) & 0x3FFFFu) >> 4;
    auto wait = [&](unsigned long long* bar, int parity) {
      return (bool)__all_sync(0xffffffffu, fa_mbar_wait(bar, (unsigned)parity));
    };
    auto wait_place = [&](int n) { return wait(&full[n % SP_BUFFERS], (n / SP_BUFFERS) & 1); };
    auto scores = [&](int l, int b) {
      const int buf = k_place(block_of(l, b)) % SP_BUFFERS;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const unsigned a_at = q_at + (unsigned)((split ? 0 : l) * (kTileBytes >> 4));
      const unsigned b_at = ring_at + (unsigned)(buf * (kTileBytes >> 4));
      const unsigned s_t = tmem_base + (unsigned)(l * 128);
      if (leader) {
#pragma unroll 1
        for (int kk = 0; kk < HEAD_DIM / 16; ++kk) {
          const unsigned off = (unsigned)((kk / 4) * (kSubTile >> 4) + 2 * (kk % 4));
          fa_mma(s_t, a_at + off, b_at + off, idesc_s, kk != 0);
        }
        fa_commit(&s_full[l]);
        if (split || l == 1) fa_commit(&empty[buf]);
      }
      __syncwarp();
    };
    bool ok = wait(q_full, 0);
    for (int l = 0; ok && l < 2; ++l)
      if (steps_of(l) > 0 && (ok = wait_place(k_place(block_of(l, 0))))) scores(l, 0);
    const int most = steps_of(0);
    for (int b = 0; ok && b < most; ++b) {
      for (int l = 0; ok && l < 2; ++l) {
        if (b >= steps_of(l)) continue;
        const int place = v_place(block_of(l, b)), buf = place % SP_BUFFERS;
        ok = wait_place(place) && wait(&p_ready[l], b & 1);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned p_t = tmem_base + (unsigned)(kPFirst + l * 128), o_t = tmem_base + 256u + (unsigned)(l * 128);
        const unsigned b_at = ring_at + (unsigned)(buf * (kTileBytes >> 4));
        if (leader) {
#pragma unroll 1
          for (int kk = 0; kk < SP_KEYS / 16; ++kk)
            fa_mma_ts(o_t, p_t + (unsigned)(kk * 8), b_at + (unsigned)(kk * 128), idesc_o, b > 0 || kk != 0);
          fa_commit(&pv_done[l]);
          if (split || l == 1) fa_commit(&empty[buf]);
        }
        __syncwarp();
        if (b + 1 < steps_of(l)) {
          ok = wait_place(k_place(block_of(l, b + 1))) && (!kPOnScores || wait(&pv_done[l], b & 1));
          if (ok) scores(l, b + 1);
        }
      }
    }
  } else if (live && warp < SP_SOFTMAX_WARPS) {
    // ---------------- softmax: two threads a row, 64 of a block's keys each ----------------
    const int l = warp >> 3, half = (warp >> 2) & 1;
    const int r = (warp & 3) * 32 + lane;
    const unsigned lane_base = ((unsigned)((warp & 3) * 32) << 16);
    const unsigned my_s = tmem_base + lane_base + (unsigned)(l * 128);
    const unsigned my_p = my_s + (unsigned)(kPFirst + half * (kHalfKeys / 2));
    const unsigned my_o = my_s + 256u;
    float* my_stat = stat_s + (l * 2 + half) * SP_ROWS + r;
    const float* other_stat = stat_s + (l * 2 + 1 - half) * SP_ROWS + r;
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + l * 4 + (warp & 3)) : "memory"); };
    int row = r < rows_of(l) ? member_of(l, r) : -1;
    if (row >= n_rows) {
      tokb200_report_error(TOKB200_LIB_SHARED_PREFIX_TCGEN05, 3);
      row = -1;
    }
    if (!split || l == 0) {
      // the rows of q that the warp's lanes own, half of a row's lanes a warp, 16 bytes a load; behind the members: zeros
      constexpr int kPieces = HEAD_DIM / 16, kRowsAtOnce = 32 / kPieces;
      uint4 v[32 / kRowsAtOnce];
#pragma unroll
      for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
        const int in_warp = i * kRowsAtOnce + lane / kPieces, from = __shfl_sync(0xffffffffu, row, in_warp);
        const int head = kvh * group + ((warp & 3) * 32 + in_warp) % group;
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (from >= 0) v[i] = *reinterpret_cast<const uint4*>(q + ((size_t)from * nh + head) * HEAD_DIM + (half * kPieces + lane % kPieces) * 8);
      }
#pragma unroll
      for (int i = 0; i < 32 / kRowsAtOnce; ++i) {
        const int at = (warp & 3) * 32 + i * kRowsAtOnce + lane / kPieces, c = half * kPieces + lane % kPieces;
        *reinterpret_cast<uint4*>(q_s + l * kTileBytes + (c / 8) * kSubTile + swz(at, c % 8)) = v[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    if (lane == 0) fa_mbar_arrive(q_full);
    const int steps = steps_of(l);
    float m_ref = -INFINITY, l_run = 0.f;     // reference maximum (raw score units, the row's) and running sum (this half's)
    bool ok = true;
    for (int b = 0; b < steps; ++b) {
      const int kb = first + block_of(l, b) * SP_KEYS + half * kHalfKeys;
      // behind a wait that ran out a warp goes on through its steps without waiting, so that it meets its partner as often as
      // that one does
      ok = __all_sync(0xffffffffu, ok && fa_mbar_wait(&s_full[l], b & 1));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float s[kHalfKeys];
      fa_tmem_load64(my_s + (unsigned)(half * kHalfKeys), s);
      if (CAPPED) {
#pragma unroll
        for (int j = 0; j < kHalfKeys; ++j) s[j] = softcap_raw(s[j], cap_in, cap_out);
      }
      if (kb + kHalfKeys > end) {
#pragma unroll
        for (int j = 0; j < kHalfKeys; ++j) s[j] = kb + j < end ? s[j] : -INFINITY;
      }
      float m8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m8[i] = fmaxf(s[i], s[8 + i]);
#pragma unroll
      for (int j = 16; j < kHalfKeys; j += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(m8[i], s[j + i]);
      float m_blk = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
      *my_stat = m_blk;
      if (kPOnScores) asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      meet();
      if (kPOnScores) asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      m_blk = fmaxf(m_blk, *other_stat);
      const bool move = m_blk > -INFINITY && (m_ref == -INFINITY || (m_blk - m_ref) * scale_log2 > SP_RESCALE_AT);
      float factor = 1.f;
      if (move) {
        factor = m_ref == -INFINITY ? 0.f : fa_exp2((m_ref - m_blk) * scale_log2);
        m_ref = m_blk;
        l_run *= factor;
      }
      const float m_scaled = m_ref == -INFINITY ? 0.f : m_ref * scale_log2;
      const unsigned long long scale2 = fa_pack2(scale_log2, scale_log2), shift2 = fa_pack2(-m_scaled, -m_scaled);
      unsigned long long sum2[4] = {0ull, 0ull, 0ull, 0ull};
      unsigned p[kHalfKeys / 2];
#pragma unroll
      for (int j = 0; j < kHalfKeys; j += 2) {
        float x0, x1;
        fa_unpack2(fa_fma2(fa_pack2(s[j], s[j + 1]), scale2, shift2), x0, x1);
        x0 = fa_exp2(x0);
        x1 = fa_exp2(x1);
        sum2[(j >> 1) & 3] = fa_add2(sum2[(j >> 1) & 3], fa_pack2(x0, x1));
        const __nv_bfloat162 pair = __floats2bfloat162_rn(x0, x1);
        p[j >> 1] = *reinterpret_cast<const unsigned*>(&pair);
      }
      float sum_even, sum_odd;
      fa_unpack2(fa_add2(fa_add2(sum2[0], sum2[1]), fa_add2(sum2[2], sum2[3])), sum_even, sum_odd);
      l_run += sum_even + sum_odd;
      fa_tmem_store32(my_p, p);
      if (b > 0 && __any_sync(0xffffffffu, move)) {
        ok = __all_sync(0xffffffffu, ok && fa_mbar_wait(&pv_done[l], (b - 1) & 1));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
        for (int c0 = half * (HEAD_DIM / 2); c0 < (half + 1) * (HEAD_DIM / 2); c0 += 16) {
          float acc[16];
          fa_tmem_load16(my_o + (unsigned)c0, acc);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[j] *= factor;
          fa_tmem_store16(my_o + (unsigned)c0, acc);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (ok && lane == 0) fa_mbar_arrive(&p_ready[l]);                    // one arrival a warp
    }
    // ---------------- the row's part ----------------
    if (steps > 0) ok = ok && fa_mbar_wait(&pv_done[l], (steps - 1) & 1);
    const int other_steps = split ? steps_of(1 - l) : 0;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    *my_stat = l_run;                        // both halves' sums (the maxima were read before the last P V)
    meet();
    const float l_all = l_run + *other_stat;
    float m_all = m_ref, weight = 1.f, weight_other = 0.f, den = l_all;
    if (split) {
      meet();                                // read before the slots are written again
      *my_stat = half ? l_all : m_ref;
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      asm volatile("bar.sync 9, %0;" ::"n"(SP_SOFTMAX_WARPS * 32) : "memory");
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const float m_other = stat_s[(1 - l) * 2 * SP_ROWS + r], l_other = stat_s[((1 - l) * 2 + 1) * SP_ROWS + r];
      m_all = fmaxf(m_ref, m_other);
      weight = m_ref == -INFINITY ? 0.f : fa_exp2((m_ref - m_all) * scale_log2);
      weight_other = m_other == -INFINITY ? 0.f : fa_exp2((m_other - m_all) * scale_log2);
      den = (steps > 0 ? weight * l_all : 0.f) + (other_steps > 0 ? weight_other * l_other : 0.f);
    }
    // The part leaves through the ring's memory (both lanes' products have read all of it), a thread's run of a row in one bulk
    // copy: stored from registers, 16 bytes a row and instruction, 256 rows took 4 us.
    if (!split) asm volatile("bar.sync 9, %0;" ::"n"(SP_SOFTMAX_WARPS * 32) : "memory");
    if (__all_sync(0xffffffffu, ok)) {
      // a thread writes its half of the head; split, its quarter, from both accumulators (one without a step was never written)
      const int width = split ? HEAD_DIM / 4 : HEAD_DIM / 2, from = (split ? l * 2 + half : half) * width;
      const size_t at = ((size_t)max(row, 0) * nh + kvh * group + r % group) * pieces + piece;
      if (row >= 0 && half == 0 && (!split || l == 0)) stat_parts[at] = make_float2(m_all * scale_log2, den);
      unsigned char* out_row = ring + (split ? r : l * SP_ROWS + r) * kOutStride;
#pragma unroll 1
      for (int c0 = from; c0 < from + width; c0 += 16) {
        float acc[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.f;
        if (steps > 0) {
          float part[16];
          fa_tmem_load16(my_o + (unsigned)c0, part);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i] = weight * part[i];
        }
        if (other_steps > 0) {
          float part[16];
          fa_tmem_load16(tmem_base + lane_base + 256u + (unsigned)((1 - l) * 128 + c0), part);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[i] = fmaf(weight_other, part[i], acc[i]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<float4*>(out_row + (c0 + 4 * c) * 4) = make_float4(acc[4 * c], acc[4 * c + 1], acc[4 * c + 2], acc[4 * c + 3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      if (row >= 0)
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                     ::"l"(acc_parts + at * HEAD_DIM + from), "r"(fa_smem(out_row + from * 4)), "r"(width * 4) : "memory");
      asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group 0;" ::: "memory");
    }
  }
  // ---------------- common exit ----------------
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0 && tmem_slot[1] != 0) {
    atomicExch(&sp_error_flag, 1);
    tokb200_report_error(TOKB200_LIB_SHARED_PREFIX_TCGEN05, 1);
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((unsigned)kTmemCols) : "memory");
  }
}

// ---- the own keys, and the join ----------------------------------------------------------------------------------------
#define OWN_WARPS 4
#define OWN_THREADS (OWN_WARPS * 32)
#define OWN_TILE 32                   // keys a warp takes a turn
#define OWN_MAX_GROUP 16              // heads of a group: the rows of one mma
#define OWN_MAX_CLUSTER 8
constexpr int kSteps = HEAD_DIM / 32;                // steps of 32 lanes of the head: one 16-byte load, two mma
constexpr int kOwnStride = HEAD_DIM + 8;             // elements between staged rows of keys and of values
constexpr int kRow = HEAD_DIM + 4;                   // a part in shared memory: weighted values, maximum (log2 units), sum

__device__ __forceinline__ void own_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void own_ldmatrix_x4_trans(unsigned (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(fa_smem(p)));
}
__device__ __forceinline__ unsigned own_pack(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<unsigned*>(&v);
}
__device__ __forceinline__ void own_cluster_sync() {
  __syncwarp();                                      // the barrier wants a warp whole, whatever loop it comes from
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// four floats of block `rank` of this cluster, at the place `local` has in this block's shared memory (no memory clobber: several
// may be on their way)
__device__ __forceinline__ float4 own_peer(const float* local, unsigned rank) {
  unsigned theirs;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"(fa_smem(local)), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(theirs));
  return v;
}
// lanes of the head that thread t of a quad reads in step st: a permutation that q and keys share, which a dot product does
// not see; a quad's two pieces of 16 bytes lie side by side
__device__ __forceinline__ int own_lane(int st, int t) { return (st >> 1) * 64 + 16 * t + 8 * (st & 1); }

// `alone`: no first kernel runs in front of this one
__global__ void __launch_bounds__(OWN_THREADS, 3)
shared_prefix_own_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k_pool,
                         const __nv_bfloat16* __restrict__ v_pool, __nv_bfloat16* __restrict__ out,
                         const int* __restrict__ block_table, int table_stride, const int* __restrict__ row_req,
                         const int* __restrict__ pos, const int* __restrict__ shared, int nh, int nkv, int page, int tile_pieces,
                         float scale, const float* __restrict__ sink, float softcap, int alone, const float* __restrict__ acc_parts,
                         const float2* __restrict__ stat_parts) {
  const int rank = blockIdx.x, size = gridDim.x, kvh = blockIdx.y, row = blockIdx.z;
  const int group = nh / nkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  if (alone) pdl_wait();
  const int req = row_req[row];
  if (req < 0) {                                     // the same for the whole cluster
    if (!alone) pdl_wait();
    pdl_launch();
    return;
  }
  const int reach = table_stride * page, common = shared ? min(max(shared[row], 0), reach) : 0;
  const int n_own = max(min(pos[row] + 1, reach) - common, 0);
  const int len = ((n_own + size - 1) / size + OWN_TILE - 1) / OWN_TILE * OWN_TILE;
  const int first = common + rank * len, last = common + min(n_own, (rank + 1) * len) - 1;     // none: last < first
  const int n_tile = common > 0 ? (common + sp_piece(common, tile_pieces) - 1) / sp_piece(common, tile_pieces) : 0;
  const int* table = block_table + (size_t)req * table_stride;
  __nv_bfloat16* k_s = reinterpret_cast<__nv_bfloat16*>(fa_raw) + (size_t)warp * 2 * OWN_TILE * kOwnStride;
  __nv_bfloat16* v_s = k_s + OWN_TILE * kOwnStride;

  const int page_shift = (page & (page - 1)) == 0 ? __ffs(page) - 1 : -1;
  auto tile_slots = [&](int k0) {                    // a key a lane
    const int key = k0 + lane;
    if (key > last) return -1;
    const int pg = page_shift >= 0 ? key >> page_shift : key / page;
    return max(table[pg], 0) * page + (key - pg * page);
  };
  // a tile's rows, 16 bytes a copy, a row's pieces side by side; rows behind the last key: zeros
  auto stage = [&](int my_slot, const __nv_bfloat16* pool, __nv_bfloat16* dst_rows) {
    constexpr int kPieces = HEAD_DIM / 8;
#pragma unroll
    for (int c = 0; c < kPieces; ++c) {
      const int i = c * 32 + lane, at = i / kPieces, piece = i % kPieces;
      const int slot = __shfl_sync(0xffffffffu, my_slot, at);
      fa_copy16(dst_rows + at * kOwnStride + piece * 8, pool + ((size_t)max(slot, 0) * nkv + kvh) * HEAD_DIM + piece * 8, slot >= 0);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  const int k_mine = first + warp * OWN_TILE;
  if (k_mine <= last) {
    const int slots = tile_slots(k_mine);
    stage(slots, k_pool, k_s);
    stage(slots, v_pool, v_s);
  }
  unsigned qa[kSteps][2][4];
  {
    const __nv_bfloat16* qa_row = q + ((size_t)row * nh + kvh * group + g) * HEAD_DIM;
    const __nv_bfloat16* qb_row = qa_row + (size_t)8 * HEAD_DIM;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
      const uint4 a = g < group ? *reinterpret_cast<const uint4*>(qa_row + own_lane(st, t)) : none;
      const uint4 b = g + 8 < group ? *reinterpret_cast<const uint4*>(qb_row + own_lane(st, t)) : none;
      qa[st][0][0] = a.x; qa[st][0][1] = b.x; qa[st][0][2] = a.y; qa[st][0][3] = b.y;
      qa[st][1][0] = a.z; qa[st][1][1] = b.z; qa[st][1][2] = a.w; qa[st][1][3] = b.w;
    }
  }
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  float o[HEAD_DIM / 8][4];
#pragma unroll
  for (int i = 0; i < HEAD_DIM / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const float scale_log2 = scale * 1.4426950408889634f;
  const bool capped = softcap > 0.f;
  const float cap_in = capped ? scale / softcap : 0.f, cap_out = softcap * 1.4426950408889634f;
#pragma unroll 1
  for (int k0 = k_mine; k0 <= last; k0 += OWN_WARPS * OWN_TILE) {
    const int k_next = k0 + OWN_WARPS * OWN_TILE;
    const bool more = k_next <= last;
    const int slots_next = more ? tile_slots(k_next) : -1;
    asm volatile("cp.async.wait_group 1;\n" ::: "memory");     // this tile's keys have landed (its values may not)
    __syncwarp();
    float s[OWN_TILE / 8][4];
#pragma unroll
    for (int nt = 0; nt < OWN_TILE / 8; ++nt) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
      const __nv_bfloat16* k_row = k_s + (nt * 8 + g) * kOwnStride;
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const uint4 kf = *reinterpret_cast<const uint4*>(k_row + own_lane(st, t));
        own_mma(s[nt], qa[st][0], kf.x, kf.y);
        own_mma(s[nt], qa[st][1], kf.z, kf.w);
      }
    }
    __syncwarp();
    if (more) stage(slots_next, k_pool, k_s);
    float m_new[2] = {m_run[0], m_run[1]};
#pragma unroll
    for (int nt = 0; nt < OWN_TILE / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = capped ? softcap_raw(s[nt][e], cap_in, cap_out) : s[nt][e] * scale_log2;
        s[nt][e] = k0 + nt * 8 + 2 * t + (e & 1) <= last ? x : -INFINITY;
        m_new[e >> 1] = fmaxf(m_new[e >> 1], s[nt][e]);
      }
    float corr[2], base[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m_new[i] = fmaxf(m_new[i], __shfl_xor_sync(0xffffffffu, m_new[i], 1));
      m_new[i] = fmaxf(m_new[i], __shfl_xor_sync(0xffffffffu, m_new[i], 2));
      base[i] = m_new[i] == -INFINITY ? 0.f : m_new[i];
      corr[i] = exp2f(m_run[i] - base[i]);                                   // 0 on the first turn
      m_run[i] = m_new[i];
    }
#pragma unroll
    for (int nt = 0; nt < OWN_TILE / 8; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = exp2f(s[nt][e] - base[e >> 1]);
        s[nt][e] = p;
        sum[e >> 1] += p;
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      l_run[i] = l_run[i] * corr[i] + sum[i];
    }
#pragma unroll
    for (int i = 0; i < HEAD_DIM / 8; ++i) {
      o[i][0] *= corr[0]; o[i][1] *= corr[0];
      o[i][2] *= corr[1]; o[i][3] *= corr[1];
    }
    if (more) asm volatile("cp.async.wait_group 1;\n" ::: "memory");   // this tile's values have landed (the next keys may not)
    else asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncwarp();
#pragma unroll
    for (int ks = 0; ks < OWN_TILE / 16; ++ks) {
      unsigned pf[4];
      pf[0] = own_pack(s[2 * ks][0], s[2 * ks][1]);
      pf[1] = own_pack(s[2 * ks][2], s[2 * ks][3]);
      pf[2] = own_pack(s[2 * ks + 1][0], s[2 * ks + 1][1]);
      pf[3] = own_pack(s[2 * ks + 1][2], s[2 * ks + 1][3]);
#pragma unroll
      for (int dp = 0; dp < HEAD_DIM / 16; ++dp) {
        unsigned vf[4];
        own_ldmatrix_x4_trans(vf, v_s + (ks * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * kOwnStride + dp * 16 + (lane >> 4) * 8);
        own_mma(o[2 * dp], pf, vf[0], vf[1]);
        own_mma(o[2 * dp + 1], pf, vf[2], vf[3]);
      }
    }
    __syncwarp();
    if (more) stage(slots_next, v_pool, v_s);
  }

  // ---- the block's part: its warps' joined (the buffer takes the place of the staged values) ----
  __syncthreads();
  float* acc_s = reinterpret_cast<float*>(fa_raw);               // [warp][head][kRow]
  float* piece_s = acc_s + (size_t)OWN_WARPS * group * kRow;     // [head][kRow]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int head = g + 8 * i;
    if (head < group) {
      float* dst = acc_s + ((size_t)warp * group + head) * kRow;
#pragma unroll
      for (int nt = 0; nt < HEAD_DIM / 8; ++nt) *reinterpret_cast<float2*>(dst + nt * 8 + 2 * t) = make_float2(o[nt][2 * i], o[nt][2 * i + 1]);
      if (t == 0) *reinterpret_cast<float2*>(dst + HEAD_DIM) = make_float2(m_run[i], l_run[i]);
    }
  }
  __syncthreads();
  for (int i = tid; i < group * HEAD_DIM; i += OWN_THREADS) {
    const int head = i / HEAD_DIM, c = i % HEAD_DIM;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < OWN_WARPS; ++w) m = fmaxf(m, acc_s[((size_t)w * group + head) * kRow + HEAD_DIM]);
    const float base = m == -INFINITY ? 0.f : m;                 // no warp has keys: a part of nothing
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < OWN_WARPS; ++w) {
      const float* src = acc_s + ((size_t)w * group + head) * kRow;
      const float f = exp2f(src[HEAD_DIM] - base);               // a warp without keys: 0
      num += f * src[c];
      den += f * src[HEAD_DIM + 1];
    }
    piece_s[(size_t)head * kRow + c] = num;
    if (c == 0) { piece_s[(size_t)head * kRow + HEAD_DIM] = m; piece_s[(size_t)head * kRow + HEAD_DIM + 1] = den; }
  }
  if (size > 1) own_cluster_sync(); else __syncthreads();
  if (!alone) pdl_wait();                            // the parts of the common keys are there
  pdl_launch();
  // ---- every size-th head of the group, half a warp each: the pieces of the cluster's blocks and the parts of the common keys ----
  const int n_parts = size + n_tile, hl = lane & 15;
  for (int i0 = 2 * warp; rank + size * i0 < group; i0 += 2 * OWN_WARPS) {
    const int head = rank + size * (i0 + (lane >> 4));
    const bool on = head < group;
    const float* piece = piece_s + (size_t)(on ? head : 0) * kRow;
    const size_t at = ((size_t)row * nh + kvh * group + (on ? head : 0)) * tile_pieces;
    // two parts a lane: their maxima, sums and weights
    float m[2], l[2], f[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = hl + 16 * e;
      m[e] = -INFINITY;
      l[e] = 0.f;
      if (i < size) {
        const float4 v = size > 1 ? own_peer(piece + HEAD_DIM, (unsigned)i) : *reinterpret_cast<const float4*>(piece + HEAD_DIM);
        m[e] = v.x;
        l[e] = v.y;
      } else if (i < n_parts) {
        const float2 v = __ldcg(&stat_parts[at + i - size]);
        m[e] = v.x;
        l[e] = v.y;
      }
    }
    float m_all = fmaxf(m[0], m[1]), den = 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      f[e] = exp2f(m[e] - m_all);
      den += hl + 16 * e < n_parts ? f[e] * l[e] : 0.f;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    if (sink && on) den += exp2f(sink[kvh * group + head] * 1.4426950408889634f - m_all);
    constexpr int kQuads = HEAD_DIM / 64;                        // four lanes of the head at a time: hl and, of 128, hl + 16
    float num[kQuads][4] = {};
    auto weight_of = [&](int i) { return __shfl_sync(0xffffffffu, i < 16 ? f[0] : f[1], (lane & 16) | (i & 15)); };
    auto add = [&](int k, float w, const float4& v) {
      num[k][0] = fmaf(w, v.x, num[k][0]);
      num[k][1] = fmaf(w, v.y, num[k][1]);
      num[k][2] = fmaf(w, v.z, num[k][2]);
      num[k][3] = fmaf(w, v.w, num[k][3]);
    };
    if (size == 1) {
      const float w = weight_of(0);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) add(k, w, *reinterpret_cast<const float4*>(piece + (hl + 16 * k) * 4));
    } else {
      for (int i = 0; i < size; i += 2) {                        // a power of two
        float4 v[2][kQuads];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int k = 0; k < kQuads; ++k) v[e][k] = own_peer(piece + (hl + 16 * k) * 4, (unsigned)(i + e));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float w = weight_of(i + e);
#pragma unroll
          for (int k = 0; k < kQuads; ++k) add(k, w, v[e][k]);
        }
      }
    }
#pragma unroll 8
    for (int i = 0; i < n_tile; ++i) {
      const float w = weight_of(size + i);
      const float4* src = reinterpret_cast<const float4*>(acc_parts + (at + i) * HEAD_DIM);
#pragma unroll
      for (int k = 0; k < kQuads; ++k) add(k, w, __ldcg(src + hl + 16 * k));
    }
    const bool any = n_tile + n_own > 0;                         // a row without a key: zeros
    const float inv = any ? 1.0f / den : 0.f;
    __nv_bfloat16* dst = out + ((size_t)row * nh + kvh * group + head) * HEAD_DIM;
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
      if (on)
        *reinterpret_cast<uint2*>(dst + (hl + 16 * k) * 4) =
            any ? make_uint2(own_pack(num[k][0] * inv, num[k][1] * inv), own_pack(num[k][2] * inv, num[k][3] * inv)) : make_uint2(0u, 0u);
  }
  if (size > 1) own_cluster_sync();                  // nobody leaves while its piece may still be read
}

TOKB200_API int tokb200_shared_prefix_tcgen05_error(void) {
  int flag = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&flag, sp_error_flag, sizeof(int)) != cudaSuccess) return -1;
  if (flag) cudaMemcpyToSymbol(sp_error_flag, &zero, sizeof(int));
  return flag;
}

// (pieces of a tile's keys, blocks of a row's own keys) for a launch of these sizes; no tiles: the rows' whole keys are their own.
TOKB200_API int tokb200_shared_prefix_tcgen05_pieces(int n_rows, int n_tiles, int nkv, int reach, int* tile_pieces, int* own_pieces) {
  const int sms = 148, own_an_sm = 3;
  const int units = n_rows * nkv;
  int own = 1;
  while (own < OWN_MAX_CLUSTER && (n_tiles > 0 ? units * own * 2 <= sms / 2 && own * 1024 <= reach : units * own * 2 <= own_an_sm * sms && own * 128 < reach))
    own *= 2;
  *own_pieces = own;
  // the first kernel's blocks, one a multiprocessor, beside as many as the second one's take
  const int tiles = n_tiles > 0 ? n_tiles * nkv : 1, left = sms - (units * own + own_an_sm - 1) / own_an_sm, most = (reach + SP_KEYS - 1) / SP_KEYS;
  int pieces = (left > sms / 3 ? left : sms / 3) / tiles;
  if (pieces > most) pieces = most;
  *tile_pieces = pieces < 1 ? 1 : pieces > SP_MAX_PIECES ? SP_MAX_PIECES : pieces;
  return TOKB200_OK;
}

// As tokb200_shared_prefix_attention; `parts` holds n_rows * nh * tile_pieces * (HEAD_DIM + 2) floats where there are tiles.
TOKB200_API int tokb200_shared_prefix_tcgen05(
    const void* q, const void* k_pool, const void* v_pool, void* out, const int* block_table, int table_stride, const int* row_req,
    const int* pos, const int* shared, const int* members, int n_listed, const int* tiles, int n_tiles, int n_rows, int pool_rows, int nh, int nkv,
    int d, int page, float scale, const float* sink, float softcap, int tile_pieces, int own_pieces, float* parts,
    cudaStream_t stream) {
  if (n_rows <= 0) return TOKB200_OK;
  if (d != HEAD_DIM || nh <= 0 || nkv <= 0 || nh % nkv || nh / nkv > OWN_MAX_GROUP || page <= 0 || page % 8 || pool_rows <= 0 || n_tiles < 0 || n_listed < 0 ||
      n_tiles > 65535 || n_rows > 65535 || nkv > 65535 || table_stride <= 0 || (long long)table_stride * page > 0x7fffffffLL ||
      tile_pieces < 1 || tile_pieces > SP_MAX_PIECES || own_pieces < 1 || own_pieces > OWN_MAX_CLUSTER || (own_pieces & (own_pieces - 1)))
    return TOKB200_BAD_SIZE;
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out | (uintptr_t)tiles | (uintptr_t)parts) & 15)
    return TOKB200_BAD_ALIGNMENT;
  float* acc_parts = parts;                            // behind them the maxima and sums
  float2* stat_parts = (float2*)(parts + (size_t)n_rows * nh * tile_pieces * HEAD_DIM);
  const int group = nh / nkv;
  const size_t stage = (size_t)2 * OWN_WARPS * OWN_TILE * kOwnStride * sizeof(__nv_bfloat16);
  const size_t merge = (size_t)(OWN_WARPS + 1) * group * kRow * sizeof(float);
  const size_t own_smem = stage > merge ? stage : merge;
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return TOKB200_BAD_SIZE;
  if (!configured[device]) {
    cudaError_t err = cudaFuncSetAttribute(shared_prefix_tcgen05_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFaSmem);
    if (err == cudaSuccess)
      err = cudaFuncSetAttribute(shared_prefix_tcgen05_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFaSmem);
    if (err == cudaSuccess)
      err = cudaFuncSetAttribute(shared_prefix_own_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (err != cudaSuccess) return (int)err;
    configured[device] = true;
  }
  if (n_tiles > 0) {
    int run = page & -page;                            // keys that lie together in a page whatever the block, up to a block
    run = run > SP_KEYS ? SP_KEYS : run;
    CUtensorMap map_k, map_v;
    int status = fa_map(&map_k, k_pool, pool_rows, (long long)nkv * HEAD_DIM, run);
    if (status == TOKB200_OK) status = fa_map(&map_v, v_pool, pool_rows, (long long)nkv * HEAD_DIM, run);
    if (status != TOKB200_OK) return status;
    // strictly behind its predecessor, as attention_tcgen05.cu explains
    status = launch_ordered(false, softcap > 0.f ? shared_prefix_tcgen05_kernel<true> : shared_prefix_tcgen05_kernel<false>,
                            dim3(tile_pieces, nkv, n_tiles), dim3(SP_THREADS), (size_t)kFaSmem, stream, map_k, map_v, (const __nv_bfloat16*)q,
                            (const __nv_bfloat16*)v_pool, block_table, table_stride, row_req, members, n_listed, (const int4*)tiles, n_rows, nh,
                            nkv, page, run, pool_rows, tile_pieces, scale * 1.4426950408889634f, softcap > 0.f ? scale / softcap : 0.f,
                            softcap > 0.f ? softcap / scale : 0.f, acc_parts, stat_parts);
    if (status != TOKB200_OK) return status;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(own_pieces, nkv, n_rows);
  config.blockDim = dim3(OWN_THREADS);
  config.dynamicSmemBytes = own_smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = tokb200_early_starts();
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = (unsigned)own_pieces;
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t err = cudaLaunchKernelEx(&config, shared_prefix_own_kernel, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k_pool,
                                             (const __nv_bfloat16*)v_pool, (__nv_bfloat16*)out, block_table, table_stride, row_req, pos, shared,
                                             nh, nkv, page, tile_pieces, scale, sink, softcap, n_tiles > 0 ? 0 : 1, (const float*)acc_parts,
                                             (const float2*)stat_parts);
  return err == cudaSuccess ? TOKB200_OK : (int)err;
}
