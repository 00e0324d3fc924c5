// Bookkeeping of a paged KV cache on the GPU, without a word to the host (fa_b200.h says what each call does):
//   reserve_pages  block tables and slot maps from request lengths
//   release_pages  pages back on the stack of unused ones
//   tree_layout    what the nodes of drafted trees see, and their positions
//   keep_path      the accepted path of each tree moves up in the caches
// All but the last are bound by latency: a launch, a scan over the sequences, two or three loads that depend on each other.
#include "fa_common.cuh"

namespace fa {

namespace {

constexpr int kPlanThreads = 512;

// (sums that cannot run over: a wrong length must not turn into a small one)
__device__ __forceinline__ uint32_t sat_add(uint32_t x, uint32_t y) {
  const uint32_t s = x + y;  // both below 2^31
  return s > 0x7fffffffu ? 0x7fffffffu : s;
}

// Inclusive sums of two numbers per thread over the block; `carry` is what came before and moves on by the block's sum.
// (`warps`: those that hold anything)
__device__ __forceinline__ void block_scan(uint32_t& x, uint32_t& y, uint32_t (&carry)[2], uint32_t (*warp_sums)[kPlanThreads / 32], int warps) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) x = sat_add(x, u), y = sat_add(y, v);
  }
  __syncthreads();  // (the sums of the round before have been read)
  if (lane == 31) warp_sums[0][warp] = x, warp_sums[1][warp] = y;
  __syncthreads();
  uint32_t before[2] = {carry[0], carry[1]};
#pragma unroll 4
  for (int w = 0; w < warps; ++w) {
    const uint32_t u = warp_sums[0][w], v = warp_sums[1][w];
    if (w < warp) before[0] = sat_add(before[0], u), before[1] = sat_add(before[1], v);
    carry[0] = sat_add(carry[0], u), carry[1] = sat_add(carry[1], v);
  }
  x = sat_add(x, before[0]), y = sat_add(y, before[1]);
}

__device__ __forceinline__ uint32_t length_of(int n) { return n < 0 ? 0u : n > 0x3fffffff ? 0x3fffffffu : (uint32_t)n; }

// The CTA that is through last sets the number of unused pages: by then every CTA has read it.
__device__ __forceinline__ void set_num_free(int32_t* num_free, int value) {
  if (threadIdx.x != 0) return;
  if (gridDim.x > 1) {
    __threadfence();
    if (atomicAdd(num_free + 1, 1) != (int)gridDim.x - 1) return;
    num_free[1] = 0;
  }
  num_free[0] = value;
}

struct ReserveParams {
  FaReserveArgs a;
  FastDiv page, each;  // rows of a page, new tokens of a sequence where all have as many
  int32_t tokens_per_cta;
};

// Every CTA scans all sequences (their lengths are in the L2 after the first) and then fills its share of the slots and of the tables' new
// entries: one launch, nothing to wait for but the number of unused pages at the end.
__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(const __grid_constant__ ReserveParams p) {
  const FaReserveArgs& a = p.a;
  extern __shared__ int32_t plan_smem[];
  uint32_t* start = reinterpret_cast<uint32_t*>(plan_smem);             // (batch + 1) first packed row
  int32_t* first = plan_smem + a.batch + 1;                             // (batch) number of its first new page, -1: no room
  uint32_t* len = reinterpret_cast<uint32_t*>(first + a.batch);         // (batch)
  __shared__ uint32_t warp_sums[2][kPlanThreads / 32];
  __shared__ int used;
  const int tid = threadIdx.x;
  const int num_free = max(0, min(a.num_free[0], a.pool));
  if (tid == 0) used = 0, start[0] = 0;
  uint32_t carry[2] = {0, 0};
  const uint32_t ps = p.page.d;
  for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    uint32_t L = 0, n = 0, need = 0;
    bool fits = true;
    if (b < a.batch) {
      L = length_of(a.cache_seqlens[b]);
      n = length_of(a.new_lens ? a.new_lens[b] : a.new_len);
      const uint32_t have = p.page.div(L + ps - 1), want = p.page.div(L + n + ps - 1);
      fits = want <= (uint32_t)a.per_seq;
      need = fits ? want - have : 0;
    }
    uint32_t rows = n, pages = need;
    block_scan(rows, pages, carry, warp_sums, min(kPlanThreads / 32, (a.batch - b0 + 31) / 32));
    const bool room = fits && (need == 0 || pages <= (uint32_t)num_free);
    const int taken = __reduce_max_sync(0xffffffffu, room && need ? (int)pages : 0);
    if ((tid & 31) == 0 && taken) atomicMax(&used, taken);
    if (b < a.batch) {
      start[b + 1] = rows;
      first[b] = room ? (int32_t)(pages - need) : -1;
      len[b] = L;
      if (blockIdx.x == (unsigned)(b / kPlanThreads) % gridDim.x) {
        a.cu_seqlens[b + 1] = (int32_t)rows;
        if (b == 0) a.cu_seqlens[0] = 0;
        a.seqlens[b] = a.cache_seqlens[b] + (room ? (int)n : 0);
      }
    }
  }
  __syncthreads();
  const int in_use = used;
  // New entries of the tables: the first token of each page writes its entry with its slot, below.  A warp per sequence where there are more tokens than rows.
  if (start[a.batch] > (uint64_t)a.total)
    for (int b = blockIdx.x * (kPlanThreads / 32) + (tid >> 5); b < a.batch; b += gridDim.x * (kPlanThreads / 32)) {
      const int f = first[b];
      if (f < 0) continue;
      const uint32_t n = start[b + 1] - start[b], have = p.page.div(len[b] + ps - 1), want = p.page.div(len[b] + n + ps - 1);
      for (uint32_t q = have + (tid & 31); q < want; q += 32) a.block_table[b * a.table_stride + q] = a.free_pages[num_free - 1 - (f + (int)(q - have))];
    }
  // slots
  const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_cta, t1 = min(t0 + p.tokens_per_cta, a.total);
  // (four rows of a thread at a time: their loads depend on a search each, but not on one another)
  for (int64_t tb = t0 + tid; tb < t1; tb += 4 * kPlanThreads) {
    int32_t pos[4];
    const int32_t* from[4];
    int32_t* entry[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = tb + k * kPlanThreads;
      pos[k] = 0, from[k] = nullptr, entry[k] = nullptr;
      if (t >= t1 || t >= start[a.batch]) continue;
      int b;
      if (a.new_lens) {
        int lo = 0, hi = a.batch;  // the last sequence that starts at or before t
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (start[mid] <= (uint32_t)t) lo = mid; else hi = mid;
        }
        b = lo;
      } else {
        b = (int)p.each.div((uint32_t)t);
      }
      const uint32_t at = len[b] + ((uint32_t)t - start[b]), have = p.page.div(len[b] + ps - 1), q = p.page.div(at);
      const uint32_t want = p.page.div(len[b] + (start[b + 1] - start[b]) + ps - 1);
      pos[k] = (int32_t)at;
      if (first[b] < 0 || q >= want) continue;
      int32_t* in_table = a.block_table + b * a.table_stride + q;
      from[k] = q < have ? in_table : a.free_pages + (num_free - 1 - (first[b] + (int)(q - have)));
      if (q >= have && at == q * ps) entry[k] = in_table;
    }
    int32_t page[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) page[k] = from[k] ? *from[k] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t t = tb + k * kPlanThreads;
      if (t >= t1) continue;
      a.slots[t] = from[k] ? (int64_t)page[k] * ps + ((uint32_t)pos[k] - p.page.div((uint32_t)pos[k]) * ps) : -1;
      a.positions[t] = pos[k];
      if (entry[k]) *entry[k] = page[k];
    }
  }
  set_num_free(a.num_free, num_free - in_use);
}

struct ReleaseParams {
  const int32_t* table;
  int64_t table_stride;
  int32_t batch, per_seq;
  FastDiv page;
  const int32_t* lens;
  const int32_t* keep;
  int32_t* free_pages;
  int32_t pool;
  int32_t* num_free;
  int32_t lane_bits;  // 2^lane_bits threads take a sequence's pages
};

__device__ __forceinline__ void released(const ReleaseParams& p, int b, uint32_t& lo, uint32_t& hi) {
  const uint32_t L = length_of(p.lens[b]), k = min(length_of(p.keep[b]), L);
  hi = min(p.page.div(L + p.page.d - 1), (uint32_t)p.per_seq);
  lo = min(p.page.div(k + p.page.d - 1), hi);
}

__global__ void __launch_bounds__(kPlanThreads) release_kernel(const __grid_constant__ ReleaseParams p) {
  extern __shared__ int32_t plan_smem[];  // (batch) pages released before a sequence's own
  __shared__ uint32_t warp_sums[2][kPlanThreads / 32];
  const int tid = threadIdx.x;
  const int num_free = max(0, min(p.num_free[0], p.pool));
  uint32_t carry[2] = {0, 0};
  for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
    const int b = b0 + tid;
    uint32_t lo = 0, hi = 0, none = 0;
    if (b < p.batch) released(p, b, lo, hi);
    uint32_t sum = hi - lo;
    block_scan(sum, none, carry, warp_sums, min(kPlanThreads / 32, (p.batch - b0 + 31) / 32));
    if (b < p.batch) plan_smem[b] = (int32_t)(sum - (hi - lo));
  }
  __syncthreads();
  const int64_t end = (int64_t)num_free + carry[0];
  const int lanes = 1 << p.lane_bits;  // of a sequence
  for (int b = blockIdx.x * (kPlanThreads >> p.lane_bits) + (tid >> p.lane_bits); b < p.batch; b += gridDim.x * (kPlanThreads >> p.lane_bits)) {
    uint32_t lo, hi;
    released(p, b, lo, hi);
#pragma unroll 4
    for (uint32_t q = lo + (tid & (lanes - 1)); q < hi; q += lanes) {
      const int64_t at = end - 1 - (plan_smem[b] + (int64_t)(q - lo));
      if (at >= 0 && at < p.pool) p.free_pages[at] = p.table[b * p.table_stride + q];
    }
  }
  set_num_free(p.num_free, (int)min(end, (int64_t)p.pool));
}

// One CTA per tree, a thread per node: it walks up, setting the bits of its row from the last word to the first.  Words are written once
// unless the walk ends at a node that is not there.
__global__ void __launch_bounds__(256) tree_layout_kernel(const int32_t* parents, int64_t stride_b, const int32_t* lens, int nodes, int32_t* words,
                                                          int32_t* positions) {
  extern __shared__ int32_t plan_smem[];
  const int b = blockIdx.x, n_words = (nodes + 31) / 32;
  for (int i = threadIdx.x; i < nodes; i += blockDim.x) plan_smem[i] = parents[b * stride_b + i];
  const int L = lens[b];
  __syncthreads();
  for (int i = threadIdx.x; i < nodes; i += blockDim.x) {
    uint32_t* row = reinterpret_cast<uint32_t*>(words) + ((int64_t)b * nodes + i) * n_words;
    uint32_t bits = 1u << (i & 31);
    int at = i >> 5, j = i, above = 0;
    for (int w = n_words - 1; w > at; --w) row[w] = 0;
    int up;
    while ((up = plan_smem[j]) >= 0 && up < j) {
      j = up;
      ++above;
      for (; at > (j >> 5); --at, bits = 0) row[at] = bits;
      bits |= 1u << (j & 31);
    }
    const bool real = up == -1;
    if (!real)
      for (int w = 0; w < n_words; ++w) row[w] = 0;
    else
      for (; at >= 0; --at, bits = 0) row[at] = bits;
    positions[(int64_t)b * nodes + i] = real ? L + above : -1;
  }
}

// A warp per row, a ballot per word
__global__ void __launch_bounds__(128) pack_tree_mask_kernel(const uint8_t* mask, int64_t stride_b, int64_t stride_i, int64_t stride_j, FastDiv by_nodes,
                                                             int64_t rows, int nodes, int32_t* words) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  const int b = (int)by_nodes.div((uint32_t)r), i = (int)(r - (int64_t)b * nodes), n_words = (nodes + 31) / 32;
  const uint8_t* row = mask + b * stride_b + i * stride_i;
#pragma unroll 4
  for (int w = 0; w < n_words; ++w) {
    const int j = w * 32 + lane;
    const uint32_t bits = __ballot_sync(0xffffffffu, j < nodes && row[j * stride_j] != 0);
    if (lane == 0) words[r * n_words + w] = (int32_t)bits;
  }
}

constexpr int kKeepCaches = 256;  // of one launch: their pointers travel in its parameters
struct KeepParams {
  FaKeepArgs a;
  FastDiv page, per_head;  // rows of a page, pieces of a head
  int32_t pieces;          // of a row
  void* caches[kKeepCaches];
};

// A CTA moves one sequence's rows in one cache.  A thread has a piece of the row for all steps of the path, eight of them on their way at a time: a step's
// source lies at or behind its own place and behind the sources before it, so that nothing is overwritten before it has been read.
template <typename V>
__global__ void __launch_bounds__(128) keep_path_kernel(const __grid_constant__ KeepParams p, int have_caches) {
  const FaKeepArgs& a = p.a;
  extern __shared__ int64_t keep_smem[];  // (2 * depth) places of a step's source and target in the cache, in elements, -1: nothing moves
  __shared__ int count;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int L = a.cache_seqlens[b];
  const int64_t end = a.seqlens ? a.seqlens[b] : INT64_MAX;  // first row that is not the sequence's
  auto place = [&](int64_t row) -> int64_t {
    if (row < 0 || row >= a.seqlen_cache) return -1;
    int64_t slab = a.cache_batch_idx ? a.cache_batch_idx[b] : b;
    int64_t r = row;
    if (a.block_table) {
      const int q = (int)p.page.div((uint32_t)row);
      slab = a.block_table[b * a.table_stride + q];
      r = row - (int64_t)q * a.page_block_size;
    }
    return slab < 0 || slab >= a.batch_cache ? -1 : slab * a.stride_b + r * a.stride_s;
  };
  if (tid < 32) {
    int n = 0;
    for (int i0 = 0; i0 < a.depth; i0 += 32) {
      const int i = i0 + tid;
      const int node = i < a.depth ? a.path[b * a.path_stride + i] : -1, last = i > 0 && i < a.depth ? a.path[b * a.path_stride + i - 1] : -1;
      bool on = node > last && node >= 0 && node < a.nodes && (int64_t)L + node < end;
      int64_t src = -1, dst = -1;
      if (on && have_caches) {  // a node whose row, or the row it would move to, is not there was never stored: it ends the path as well
        src = place((int64_t)L + node), dst = place((int64_t)L + i);
        on = src >= 0 && dst >= 0;
      }
      const uint32_t ends = __ballot_sync(0xffffffffu, !on);
      const int more = ends ? __ffs(ends) - 1 : 32;
      if (tid < more) keep_smem[2 * i] = node != i ? src : -1, keep_smem[2 * i + 1] = dst;
      n += more;
      if (ends) break;
    }
    if (tid == 0) {
      count = n;
      if (blockIdx.y == 0 && blockIdx.z == 0 && a.new_seqlens) a.new_seqlens[b] = L + n;
    }
  }
  __syncthreads();
  const int n = count;
  if (!have_caches) return;
  constexpr int E = sizeof(V) / 2;
  uint16_t* cache = reinterpret_cast<uint16_t*>(p.caches[blockIdx.y]);
  for (int c = blockIdx.z * 128 + tid; c < p.pieces; c += gridDim.z * 128) {
    const int h = (int)p.per_head.div((uint32_t)c);
    uint16_t* col = cache + h * a.stride_h + (c - h * (int)p.per_head.d) * E;
    for (int i0 = 0; i0 < n; i0 += 8) {
      V x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k < n && keep_smem[2 * (i0 + k)] >= 0) x[k] = *reinterpret_cast<const V*>(col + keep_smem[2 * (i0 + k)]);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k < n && keep_smem[2 * (i0 + k)] >= 0) *reinterpret_cast<V*>(col + keep_smem[2 * (i0 + k) + 1]) = x[k];
    }
  }
}

// The limit of 48 KB without this counts a kernel's static shared memory as well
int plan_smem_limit(fa_host::DeviceOnce& once, const void* kernel, int bytes, const char* name) {
  return bytes > 40 * 1024 ? fa_host::raise_smem_limit(once, kernel, 224 * 1024, name) : 0;
}

template <typename V>
int launch_keep(const FaKeepArgs& a, cudaStream_t st) {
  KeepParams p;
  p.a = a;
  p.a.caches = nullptr;
  p.page = fast_div(a.block_table ? a.page_block_size : 1);
  const int per_head = a.head_dim / (int)(sizeof(V) / 2);
  p.per_head = fast_div(per_head);
  p.pieces = per_head * a.heads_k;
  const int smem = a.depth * 16;
  static fa_host::DeviceOnce once;
  if (int rc = plan_smem_limit(once, reinterpret_cast<const void*>(&keep_path_kernel<V>), smem, "keep_path_kernel")) return rc;
  for (int c0 = 0; c0 < a.n_caches || c0 == 0; c0 += kKeepCaches) {
    const int n = a.n_caches - c0 < kKeepCaches ? a.n_caches - c0 : kKeepCaches;
    for (int i = 0; i < n; ++i) p.caches[i] = a.caches[c0 + i];
    if (c0) p.a.new_seqlens = nullptr;
    const int chunks = (p.pieces + 127) / 128;
    const dim3 grid(a.batch, n > 0 ? n : 1, n > 0 ? (chunks < 64 ? chunks : 64) : 1);
    keep_path_kernel<V><<<grid, 128, smem, st>>>(p, n > 0);
    if (int rc = fa_host::check_launch("keep_path_kernel")) return rc;
  }
  return 0;
}

}  // namespace

int reserve_pages(const FaReserveArgs& a, cudaStream_t st) {
  ReserveParams p;
  p.a = a;
  p.page = fast_div(a.page_block_size);
  p.each = fast_div(a.new_len > 0 ? a.new_len : 1);
  // One CTA up to 2048 rows and 512 sequences: the counter at the end of more than one costs more than the rows
  const int sms = fa_host::sm_count();
  int64_t ctas = (a.total + 2047) / 2048;
  if (ctas < (a.batch + 511) / 512) ctas = (a.batch + 511) / 512;
  if (ctas > sms) ctas = sms;
  if (ctas < 1) ctas = 1;
  p.tokens_per_cta = (int)(((a.total + ctas - 1) / ctas + 31) / 32 * 32);
  const int smem = (3 * a.batch + 1) * 4;
  static fa_host::DeviceOnce once;
  if (int rc = plan_smem_limit(once, reinterpret_cast<const void*>(&reserve_kernel), smem, "reserve_kernel")) return rc;
  reserve_kernel<<<(unsigned)ctas, kPlanThreads, smem, st>>>(p);
  return fa_host::check_launch("reserve_kernel");
}

int release_pages(const int32_t* block_table, int64_t table_stride, int batch, int per_seq, int page, const int32_t* lens, const int32_t* keep,
                  int32_t* free_pages, int pool, int32_t* num_free, cudaStream_t st) {
  int lane_bits = 3;  // few sequences (which may have many pages): as many threads as a CTA has for each
  while (lane_bits < 9 && (batch << (lane_bits + 1)) <= kPlanThreads) ++lane_bits;
  ReleaseParams p{block_table, table_stride, batch, per_seq, fast_div(page), lens, keep, free_pages, pool, num_free, lane_bits};
  const int ctas = batch <= 64 ? 1 : (batch + 63) / 64 < 64 ? (batch + 63) / 64 : 64;
  static fa_host::DeviceOnce once;
  if (int rc = plan_smem_limit(once, reinterpret_cast<const void*>(&release_kernel), batch * 4, "release_kernel")) return rc;
  release_kernel<<<ctas, kPlanThreads, batch * 4, st>>>(p);
  return fa_host::check_launch("release_kernel");
}

int tree_layout(const int32_t* parents, int64_t stride_b, const int32_t* lens, int batch, int nodes, int32_t* words, int32_t* positions,
                cudaStream_t st) {
  const int threads = nodes < 256 ? (nodes + 31) / 32 * 32 : 256;
  tree_layout_kernel<<<batch, threads, nodes * 4, st>>>(parents, stride_b, lens, nodes, words, positions);
  return fa_host::check_launch("tree_layout_kernel");
}

int pack_tree_mask(const uint8_t* mask, int64_t stride_b, int64_t stride_i, int64_t stride_j, int batch, int nodes, int32_t* words, cudaStream_t st) {
  const int64_t rows = (int64_t)batch * nodes;
  pack_tree_mask_kernel<<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(mask, stride_b, stride_i, stride_j, fast_div(nodes), rows, nodes, words);
  return fa_host::check_launch("pack_tree_mask_kernel");
}

int keep_path(const FaKeepArgs& a, cudaStream_t st) {
  FA_REQUIRE(a.depth <= 12288, "a path has at most 12288 nodes");
  bool pieces = a.head_dim % 8 == 0 && a.stride_b % 8 == 0 && a.stride_s % 8 == 0 && a.stride_h % 8 == 0;
  for (int i = 0; i < a.n_caches; ++i) pieces = pieces && (reinterpret_cast<uintptr_t>(a.caches[i]) & 15) == 0;
  return pieces ? launch_keep<uint4>(a, st) : launch_keep<uint16_t>(a, st);
}

}  // namespace fa
