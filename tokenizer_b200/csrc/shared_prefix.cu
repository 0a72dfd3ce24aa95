// Attention of decoding rows whose caches begin with the same pages: the general kernels (any type, head size to 256 and
// page size; the tensor-core ones for bfloat16 are in shared_prefix_tcgen05.cu).
//
// A row r sees the `keys` keys of its tile, read through the table of the tile's first live member, and its own keys from
// shared[r] up to pos[r]; a row of no tile has shared[r] = 0 and sees its own alone.  With scores s = q.k * scale (capped:
// cap * tanh(s / cap)) the output is sum(exp(s) v) / (sum(exp(s)) + exp(sink)).  A softmax splits along its keys: a part with
// maximum m, sum l = sum(exp(s - m)) and weighted values a = sum(exp(s - m) v) joins others by sum(exp(m - M) a) / sum(exp(m -
// M) l), M the largest m.  So the common keys are read once a tile, for all heads of all members together, the own keys once a
// row, each cut into pieces over blocks; every piece leaves (a, m, l) in 32 bits, and a second kernel joins them.
//
// A block takes 32 (row, head) pairs, four a warp, and walks its piece 32 keys at a time: keys and values lie in shared
// memory in 32 bits; a lane has a key for the scores (of its warp's four pairs at once, 16 multiply-adds for five 16-byte
// reads of shared memory) and every 32nd lane of the head for the weighted values.  8 rows of 14 heads of 64 lanes behind
// 1,024 common keys, 32-bit: 16.8 us on the device, 2.5 a turn of 32 keys; 16 rows with 2,000 in common 27 us (232 where
// every row reads all of its keys in the general attention).
#include "common.cuh"

#define SP_WARPS 8
#define SP_THREADS (SP_WARPS * 32)
#define SP_PAIRS_WARP 4
#define SP_PAIRS (SP_WARPS * SP_PAIRS_WARP)       // (row, head) pairs of a block
#define SP_KEYS 32
#define SP_MIN_PIECE 32
#define SP_JOIN_THREADS 64
#define SP_LOG2E 1.4426950408889634f

// keys of a piece when n keys are cut into at most `pieces`
__host__ __device__ __forceinline__ int sp_piece(int n, int pieces) {
  const int len = ((n + pieces - 1) / pieces + SP_KEYS - 1) / SP_KEYS * SP_KEYS;
  return len < SP_MIN_PIECE ? SP_MIN_PIECE : len;
}

__device__ __forceinline__ float sp_warp_max(float v) {      // one instruction; NaN only if all are
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
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
    if (row >= n_rows && threadIdx.x == 0) tokb200_report_error(TOKB200_LIB_SHARED_PREFIX, 3);
    req = row < 0 || row >= n_rows ? -1 : row_req[row];
  }
  return req;
}

// parts: [row][head][tile_pieces + own_pieces][d + 2]
template <typename T, int DI>
__global__ void __launch_bounds__(SP_THREADS, DI <= 4 ? 2 : 1)
shared_prefix_parts_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool,
                           const int* __restrict__ block_table, int table_stride, const int* __restrict__ row_req,
                           const int* __restrict__ pos, const int* __restrict__ shared, const int* __restrict__ members,
                           const int4* __restrict__ tiles, int n_tiles, int tile_members, int n_listed, int n_rows, int nh, int nkv,
                           int d, int page, float scale_log2, float cap_in, float cap_out, int tile_chunks,
                           int row_chunks, int tile_pieces, int own_pieces, float* __restrict__ parts) {
  constexpr int kD = DI * 32, kStride = kD + 4;
  extern __shared__ __align__(16) float sp_smem[];
  float* q_s = sp_smem;                              // [pair][kD]
  float* k_s = q_s + SP_PAIRS * kD;                  // [key][kStride]
  float* v_s = k_s + SP_KEYS * kStride;              // [key][kD]
  float4* p_s = reinterpret_cast<float4*>(v_s + SP_KEYS * kD);      // [warp][key]: the probabilities of a warp's pairs
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // z: the tiles, each in chunks of SP_PAIRS pairs, then the rows
  const int group = nh / nkv, kvh = blockIdx.y, piece = blockIdx.x;
  const bool common = (int)blockIdx.z < n_tiles * tile_chunks;
  const int unit = common ? blockIdx.z / tile_chunks : (blockIdx.z - n_tiles * tile_chunks) / row_chunks;
  const int chunk = common ? blockIdx.z % tile_chunks : (blockIdx.z - n_tiles * tile_chunks) % row_chunks;
  pdl_wait();
  pdl_launch();
  // the block's pairs: (member, head) of a tile, or the heads of a row; its keys first..end of table `req`
  int first_member = 0, n_pairs, req, first, end, slot;
  const int row_alone = common ? -1 : unit;
  if (common) {
    const int4 tile = tiles[unit];
    if (!sp_tile_fits(tile, tile_members, n_listed)) {
      if (threadIdx.x == 0) tokb200_report_error(TOKB200_LIB_SHARED_PREFIX, 3);
      return;
    }
    first_member = tile.x;
    n_pairs = tile.y * group;
    req = sp_tile_request(tile, members, row_req, n_rows);
    const int keys = min(tile.z, table_stride * page), len = sp_piece(keys, tile_pieces);
    first = piece * len;
    end = min(keys, first + len);
    slot = piece;
  } else {
    n_pairs = group;
    req = row_req[row_alone];
    const int from = max(shared[row_alone], 0), n = min(pos[row_alone] + 1, table_stride * page) - from, len = sp_piece(max(n, 0), own_pieces);
    first = from + piece * len;
    end = from + min(max(n, 0), (piece + 1) * len);
    slot = tile_pieces + piece;
  }
  if (req < 0 || first >= end || chunk * SP_PAIRS >= n_pairs) return;
  auto row_of = [&](int pair) { return common ? members[first_member + pair / group] : row_alone; };
  int row[SP_PAIRS_WARP], head[SP_PAIRS_WARP];
#pragma unroll
  for (int i = 0; i < SP_PAIRS_WARP; ++i) {
    const int pair = chunk * SP_PAIRS + warp * SP_PAIRS_WARP + i;
    row[i] = pair < n_pairs ? row_of(pair) : -1;
    if (row[i] >= n_rows) {
      tokb200_report_error(TOKB200_LIB_SHARED_PREFIX, 3);
      row[i] = -1;
    }
    head[i] = kvh * group + pair % group;
  }
  {
    float v[SP_PAIRS_WARP][DI];
#pragma unroll
    for (int i = 0; i < SP_PAIRS_WARP; ++i)
#pragma unroll
      for (int c = 0; c < DI; ++c)
        v[i][c] = row[i] >= 0 && lane + 32 * c < d ? to_float(q[((size_t)row[i] * nh + head[i]) * d + lane + 32 * c]) : 0.f;
#pragma unroll
    for (int i = 0; i < SP_PAIRS_WARP; ++i)
#pragma unroll
      for (int c = 0; c < DI; ++c) q_s[(warp * SP_PAIRS_WARP + i) * kD + lane + 32 * c] = v[i][c];
  }
  float m_run[SP_PAIRS_WARP], l_run[SP_PAIRS_WARP], acc[SP_PAIRS_WARP][DI];
#pragma unroll
  for (int i = 0; i < SP_PAIRS_WARP; ++i) {
    m_run[i] = -INFINITY;
    l_run[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DI; ++c) acc[i][c] = 0.f;
  }
  const int* table = block_table + (size_t)req * table_stride;
  // a warp brings every eighth key of a tile; the next tile's rows are asked for while this one is computed
  constexpr int kEach = SP_KEYS / SP_WARPS;
  T k_next[kEach][DI], v_next[kEach][DI];
  auto fetch = [&](int k0) {
    int slot[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int key = k0 + e * SP_WARPS + warp;
      slot[e] = key < end ? max(table[key / page], 0) * page + key % page : -1;
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const size_t at = ((size_t)max(slot[e], 0) * nkv + kvh) * d;
#pragma unroll
      for (int c = 0; c < DI; ++c) {                 // keys that are not seen, and lanes behind the head: zeros
        const bool on = slot[e] >= 0 && lane + 32 * c < d;
        k_next[e][c] = on ? k_pool[at + lane + 32 * c] : from_float<T>(0.f);
        v_next[e][c] = on ? v_pool[at + lane + 32 * c] : from_float<T>(0.f);
      }
    }
  };
  fetch(first);
  for (int k0 = first; k0 < end; k0 += SP_KEYS) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e)
#pragma unroll
      for (int c = 0; c < DI; ++c) {
        k_s[(e * SP_WARPS + warp) * kStride + lane + 32 * c] = to_float(k_next[e][c]);
        v_s[(e * SP_WARPS + warp) * kD + lane + 32 * c] = to_float(v_next[e][c]);
      }
    __syncthreads();
    if (k0 + SP_KEYS < end) fetch(k0 + SP_KEYS);
    float part[2][SP_PAIRS_WARP] = {};               // two sums a score: half the chain of dependent additions
    const float4* k_row = reinterpret_cast<const float4*>(k_s + lane * kStride);
#pragma unroll 8
    for (int c = 0; c < kD / 4; ++c) {
      const float4 kv = k_row[c];
#pragma unroll
      for (int i = 0; i < SP_PAIRS_WARP; ++i) {
        const float4 qv = reinterpret_cast<const float4*>(q_s + (warp * SP_PAIRS_WARP + i) * kD)[c];
        part[0][i] = fmaf(qv.x, kv.x, fmaf(qv.z, kv.z, part[0][i]));
        part[1][i] = fmaf(qv.y, kv.y, fmaf(qv.w, kv.w, part[1][i]));
      }
    }
    float p[SP_PAIRS_WARP];
#pragma unroll
    for (int i = 0; i < SP_PAIRS_WARP; ++i) {
      const float s = part[0][i] + part[1][i];
      float x = cap_out > 0.f ? cap_out * tanhf(s * cap_in) : s * scale_log2;
      if (k0 + lane >= end) x = -INFINITY;
      const float m_new = fmaxf(m_run[i], sp_warp_max(x));
      // a part whose scores are all -inf so far has no weight yet (a NaN among them goes through)
      const float corr = m_new == -INFINITY ? 1.f : exp2f(m_run[i] - m_new);
      p[i] = x == -INFINITY ? 0.f : exp2f(x - m_new);
      l_run[i] = l_run[i] * corr + p[i];             // of this lane's keys
      m_run[i] = m_new;
#pragma unroll
      for (int c = 0; c < DI; ++c) acc[i][c] *= corr;
    }
    p_s[warp * SP_KEYS + lane] = make_float4(p[0], p[1], p[2], p[3]);
    __syncwarp();
#pragma unroll 8
    for (int key = 0; key < SP_KEYS; ++key) {
      const float4 pk = p_s[warp * SP_KEYS + key];
#pragma unroll
      for (int c = 0; c < DI; ++c) {
        const float v = v_s[key * kD + lane + 32 * c];
        acc[0][c] = fmaf(pk.x, v, acc[0][c]);
        acc[1][c] = fmaf(pk.y, v, acc[1][c]);
        acc[2][c] = fmaf(pk.z, v, acc[2][c]);
        acc[3][c] = fmaf(pk.w, v, acc[3][c]);
      }
    }
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < SP_PAIRS_WARP; ++i) {
    const float l_all = warp_sum(l_run[i]);
    if (row[i] < 0) continue;
    float* part = parts + (((size_t)row[i] * nh + head[i]) * (tile_pieces + own_pieces) + slot) * (d + 2);
#pragma unroll
    for (int c = 0; c < DI; ++c)
      if (lane + 32 * c < d) part[lane + 32 * c] = acc[i][c];
    if (lane == 0) { part[d] = m_run[i]; part[d + 1] = l_all; }
  }
}

// a warp a (row, head), a part a lane for the weights
template <typename T, int DI>
__global__ void __launch_bounds__(SP_JOIN_THREADS)
shared_prefix_join_kernel(const float* __restrict__ parts, const int* __restrict__ row_req, const int* __restrict__ pos,
                          const int* __restrict__ shared, int n_rows, int nh, int d, int reach, int tile_pieces, int own_pieces,
                          const float* __restrict__ sink, T* __restrict__ out) {
  pdl_wait();
  pdl_launch();
  const int pair = blockIdx.x * (SP_JOIN_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (pair >= n_rows * nh) return;
  const int row = pair / nh, head = pair % nh;
  if (row_req[row] < 0) return;
  const int from = max(shared[row], 0), keys = min(from, reach), n = max(min(pos[row] + 1, reach) - from, 0);
  const int tile_len = sp_piece(keys, tile_pieces), own_len = sp_piece(n, own_pieces);
  const int n_tile = (keys + tile_len - 1) / tile_len, n_parts = n_tile + (n + own_len - 1) / own_len;      // at most a lane each
  const float* base = parts + (size_t)pair * (tile_pieces + own_pieces) * (d + 2);
  auto part_of = [&](int i) { return base + (size_t)(i < n_tile ? i : tile_pieces + i - n_tile) * (d + 2); };
  const bool on = lane < n_parts;
  const float m_part = on ? part_of(lane)[d] : -INFINITY, l_part = on ? part_of(lane)[d + 1] : 0.f;
  const float m = warp_max(m_part), f = exp2f(m_part - m);
  float den = warp_sum(on ? f * l_part : 0.f);
  if (sink) den += exp2f(sink[head] * SP_LOG2E - m);
  float num[DI] = {};
#pragma unroll 8
  for (int i = 0; i < n_parts; ++i) {
    const float w = __shfl_sync(0xffffffffu, f, i);
    const float* part = part_of(i);
#pragma unroll
    for (int c = 0; c < DI; ++c)
      if (lane + 32 * c < d) num[c] = fmaf(w, part[lane + 32 * c], num[c]);
  }
#pragma unroll
  for (int c = 0; c < DI; ++c)
    if (lane + 32 * c < d) out[(size_t)pair * d + lane + 32 * c] = from_float<T>(n_parts ? num[c] / den : 0.f);      // a row without a key: zeros
}

// (pieces of a tile's keys, pieces of a row's own keys) for a launch of these sizes: enough blocks for the device, at most 16
TOKB200_API int tokb200_shared_prefix_pieces(int n_rows, int n_tiles, int nkv, int reach, int* tile_pieces, int* own_pieces) {
  const int most = (reach + SP_MIN_PIECE - 1) / SP_MIN_PIECE, blocks = 148 * 4;      // together at most 32: a lane each in the join
  auto cut = [&](int units) {
    int n = units > 0 ? (blocks + units - 1) / units : 1;
    n = n > 16 ? 16 : n;
    return n > most ? most : n < 1 ? 1 : n;
  };
  *tile_pieces = cut(n_tiles * nkv);
  *own_pieces = cut(n_rows * nkv);
  return TOKB200_OK;
}

template <typename T, int DI>
static int sp_launch(const void* q, const void* k_pool, const void* v_pool, void* out, const int* block_table, int table_stride,
                     const int* row_req, const int* pos, const int* shared, const int* members, int n_listed, const int* tiles, int n_tiles,
                     int tile_members, int n_rows, int nh, int nkv, int d, int page, float scale, const float* sink, float softcap,
                     int tile_pieces, int own_pieces, float* parts, cudaStream_t stream) {
  const int group = nh / nkv;
  const int members_most = n_listed < 1 ? 1 : tile_members < n_listed ? tile_members : n_listed;
  const int tile_chunks = (members_most * group + SP_PAIRS - 1) / SP_PAIRS, row_chunks = (group + SP_PAIRS - 1) / SP_PAIRS;
  const long long units = (long long)n_tiles * tile_chunks + (long long)n_rows * row_chunks;
  if (nkv > 65535 || units > 65535) return TOKB200_BAD_SIZE;
  const size_t smem = (size_t)(SP_PAIRS * DI * 32 + SP_KEYS * (DI * 32 + 4) + SP_KEYS * DI * 32 + SP_WARPS * SP_KEYS * 4) * 4;
  static bool configured[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return TOKB200_BAD_SIZE;
  if (smem > 48 * 1024 && !configured[device]) {
    cudaError_t err = cudaFuncSetAttribute(shared_prefix_parts_kernel<T, DI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) return (int)err;
    configured[device] = true;
  }
  const dim3 grid(tile_pieces > own_pieces ? tile_pieces : own_pieces, nkv, (unsigned)units);
  int status = launch_dependent(shared_prefix_parts_kernel<T, DI>, grid, dim3(SP_THREADS), smem, stream, (const T*)q, (const T*)k_pool,
                                (const T*)v_pool, block_table, table_stride, row_req, pos, shared, members, (const int4*)tiles, n_tiles,
                                tile_members, n_listed, n_rows, nh, nkv, d, page, scale * SP_LOG2E, softcap > 0.f ? scale / softcap : 0.f,
                                softcap > 0.f ? softcap * SP_LOG2E : 0.f, tile_chunks, row_chunks, tile_pieces, own_pieces, parts);
  if (status != TOKB200_OK) return status;
  constexpr int kPairs = SP_JOIN_THREADS / 32;
  return launch_dependent(shared_prefix_join_kernel<T, DI>, dim3((unsigned)((n_rows * nh + kPairs - 1) / kPairs)), dim3(SP_JOIN_THREADS), 0,
                          stream, parts, row_req, pos, shared, n_rows, nh, d, table_stride * page, tile_pieces, own_pieces, sink, (T*)out);
}

// tiles: [n_tiles][4] = (first place in `members`, members, keys, 0); at most `tile_members` members each, out of `n_listed`.  A tile
// that is not so, or a member that is not a row, computes nothing and sets the error word.
TOKB200_API int tokb200_shared_prefix_attention(
    const void* q, const void* k_pool, const void* v_pool, void* out, int dtype, const int* block_table, int table_stride,
    const int* row_req, const int* pos, const int* shared, const int* members, int n_listed, const int* tiles, int n_tiles,
    int tile_members, int n_rows, int nh, int nkv, int d, int page, float scale, const float* sink, float softcap, int tile_pieces, int own_pieces,
    float* parts, cudaStream_t stream) {
  if (n_rows <= 0) return TOKB200_OK;
  if (nh <= 0 || nkv <= 0 || nh % nkv || d <= 0 || d > 256 || page <= 0 || n_tiles < 0 || n_listed < 0 || tile_members < 1 || tile_pieces < 1 || own_pieces < 1 ||
      tile_pieces > 65535 || table_stride <= 0 || (long long)table_stride * page > 0x7fffffffLL || (long long)n_rows * nh > 0x7fffffffLL)
    return TOKB200_BAD_SIZE;
  if ((uintptr_t)tiles & 15) return TOKB200_BAD_ALIGNMENT;
#define SP_CASE(T, DI)                                                                                                             \
  return sp_launch<T, DI>(q, k_pool, v_pool, out, block_table, table_stride, row_req, pos, shared, members, n_listed, tiles, n_tiles, \
                          tile_members, n_rows, nh, nkv, d, page, scale, sink, softcap, tile_pieces, own_pieces, parts, stream)
#define SP_TYPE(T)                                                                                                                 \
  do {                                                                                                                             \
    if (d <= 32) SP_CASE(T, 1);                                                                                                    \
    if (d <= 64) SP_CASE(T, 2);                                                                                                    \
    if (d <= 128) SP_CASE(T, 4);                                                                                                   \
    SP_CASE(T, 8);                                                                                                                 \
  } while (0)
  if (dtype == TOKB200_F32) SP_TYPE(float);
  if (dtype == TOKB200_BF16) SP_TYPE(__nv_bfloat16);
  return TOKB200_BAD_DTYPE;
}
