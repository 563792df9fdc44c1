// Attention of a few new tokens a group over the paged cache, where the tokens of a group share pages: the beams of one
// prompt (the prompt's pages in common, pages of their own behind them), or the tokens of a short chunk that is appended to
// one sequence (all pages in common, each token sees up to itself). A page is read once for all tokens of the group that have
// it and all query heads of the key/value head.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  over the positions j <= position of the token's own
//   table row (and j > position - window). A token at position -1 sees nothing: zeros.
//
// A group's query rows (tokens x query heads of one kv head, in that order) are cut into tiles. What a tile has to read is
// a list of pages: those in common, then the tokens' own, each once for the tokens that have it. The list is cut into
// `splits` stretches of equal length, a block each, so that the device is filled whatever the contexts are; running maximum
// and sum are kept in float32. Up to eight blocks form a cluster and add their results up through distributed shared memory; where there
// are more clusters, theirs go to scratch, and of the blocks that have written the same rows of it the last (a ticket;
// nobody waits) joins them in order.
//
// bfloat16, head sizes that are multiples of 16: from 64 to 128 on the 5th-generation tensor cores (namespace t5), below
// with mma.sync (mma_kernel). Probabilities are rounded to bfloat16 there, since both operands of the second product have the
// values' type: results are 0.0019 to 0.0021 (relative, root mean square) from 64 bits, where only their own rounding would leave
// 0.0017. Everything else (float32, other head sizes): fused multiply-adds on pages in shared memory (fma_kernel).
//
// A masked key has weight 0 by selection, not by arithmetic, and its value is not multiplied: a NaN or infinity in a place
// that a token does not see leaves it alone. (Products on the tensor cores multiply zeros too: pages that some row
// sees in part are looked at, and one with a value that is not finite is added element by element.)
#include "tcgen05.cuh"

namespace {
typedef __nv_bfloat16 bf16;
constexpr int PAGE = 64;
constexpr int MAX_ROWS = 128;   // query rows of a tile at most, so tokens too
constexpr int LIST = 256;       // pages listed at a time
constexpr int MAX_CLUSTER = 8, MAX_CLUSTERS = 32;
constexpr int FULL = 0x7fffffff;
constexpr int TOO_MANY = 51;    // status: a group has more tokens than the launch was told

struct Args {
  void* out;
  const void* q;
  KvLayout cache;
  const int *slots, *positions, *cuts, *shared;
  float* scratch;      // [tile, kv head][cluster][ROWS][head_dim], then [..][ROWS][2]
  unsigned* tickets;   // one a (tile, kv head) and block of a cluster, zero between launches
  int* status;
  int heads, window, tiles, splits, cluster;  // blocks of a tile and kv head; of a cluster
  int tokens, max_rows;
  float scale;
};

// What a tile's block works on: the same in every block of the tile.
struct Plan {
  int token0, tokens;            // the tile's tokens
  int row0, rows;                // its query rows, counted from the group's first
  int shared_first, shared_count, total;
  int longest;                   // the token that sees furthest: its table row names the pages in common
  int all_from, all_to;          // positions that every token sees (of those that see any)
  int position[MAX_ROWS], low[MAX_ROWS], slot[MAX_ROWS];   // of each token: it sees low .. position
  // The pages behind those in common, each once: page, index in the table row, which tokens have it (a bit each, all bits:
  // everybody). Only where the tile has at most 32 tokens and they fit; else (listed -1) a token's pages follow one
  // another: list_index has each token's first own page, list_page its place in the list.
  int listed, list_page[LIST], list_index[LIST];
  unsigned list_who[LIST];
  int last;
};

// Fills the plan (all threads call; ends with a barrier).
__device__ __forceinline__ void make_plan(Plan& p, const Args& a, int rows_per_tile) {
  const int group = blockIdx.z / a.tiles, tile = blockIdx.z % a.tiles;
  const int per_kv = a.heads / a.cache.kv_heads;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    constexpr int EACH = MAX_ROWS / 32;
    const int row0 = tile * rows_per_tile, t0 = row0 / per_kv;
    // Groups mostly have all the same number of tokens: where this one's would lie then is asked for beside the cuts.
    const int guess = group * a.max_rows;
    int pos[EACH], slot[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const int t = guess + t0 + lane + 32 * u;
      const bool there = lane + 32 * u < a.max_rows && t < a.tokens;
      pos[u] = there ? a.positions[t] : -1;
      slot[u] = there ? a.slots[t] : -1;
    }
    const int first = a.cuts[group], count = a.cuts[group + 1] - first, shared = a.shared[group];
    const int rows = min(rows_per_tile, count * per_kv - row0);
    if (lane == 0) {
      if (tile == a.tiles - 1 && count * per_kv > a.tiles * rows_per_tile)
        *reinterpret_cast<volatile int*>(a.status) = TOO_MANY;  // (the launch was made for fewer tokens a group)
      p.rows = max(rows, 0);
      p.total = 0;
    }
    if (rows > 0) {
      const int tokens = (row0 + rows - 1) / per_kv - t0 + 1;
      int furthest = -1, which = 0, least_first = FULL, from = 0, to = FULL;
      int low[EACH], pages[EACH];
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int t = lane + 32 * u;
        if (first != guess || t >= a.max_rows) {
          pos[u] = t < tokens ? a.positions[first + t0 + t] : -1;
          slot[u] = t < tokens ? a.slots[first + t0 + t] : -1;
        } else if (t >= tokens) {
          pos[u] = slot[u] = -1;
        }
      }
#pragma unroll
      for (int u = 0; u < EACH; ++u) {
        const int t = lane + 32 * u;
        if (slot[u] < 0) { slot[u] = 0; pos[u] = -1; }
        pos[u] = min(pos[u], a.cache.max_pages * PAGE - 1);
        low[u] = a.window > 0 ? max(0, pos[u] + 1 - a.window) : 0;
        pages[u] = pos[u] < 0 ? 0 : pos[u] / PAGE + 1;
        if (t < tokens) {
          p.position[t] = pos[u];
          p.low[t] = low[u];
          p.slot[t] = slot[u];
        }
        if (pos[u] >= 0) {  // (what a token that sees nothing gets is set aside at the end)
          from = max(from, low[u]);
          to = min(to, pos[u]);
          least_first = min(least_first, low[u] / PAGE);
          if (pos[u] > furthest) { furthest = pos[u]; which = t; }
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        int f = __shfl_xor_sync(0xffffffffu, furthest, o), w = __shfl_xor_sync(0xffffffffu, which, o);
        if (f > furthest || (f == furthest && w < which)) { furthest = f; which = w; }
        least_first = min(least_first, __shfl_xor_sync(0xffffffffu, least_first, o));
        from = max(from, __shfl_xor_sync(0xffffffffu, from, o));
        to = min(to, __shfl_xor_sync(0xffffffffu, to, o));
      }
      const int all = furthest < 0 ? 0 : furthest / PAGE + 1, common = min(max(shared, 0), all);
      const int shared_count = max(0, common - least_first);
      int total = shared_count, listed = -1;
      if (tokens <= 32) {
        // a lane a token, eight indexes of the table rows at a time: tokens with the same page share an entry
        const unsigned everybody = __ballot_sync(0xffffffffu, pages[0] > 0);
        listed = 0;
        for (int i0 = max(common, least_first); i0 < all && listed >= 0; i0 += 8) {
          int page[8];
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int i = i0 + n;
            const bool has = i < pages[0] && i >= low[0] / PAGE;
            page[n] = has ? a.cache.page_table[(size_t)slot[0] * a.cache.max_pages + i] : -1 - lane;
          }
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int i = i0 + n;
            const bool has = i < pages[0] && i >= low[0] / PAGE;
            const unsigned same = __match_any_sync(0xffffffffu, page[n]);
            const bool leads = has && (same & ((1u << lane) - 1u)) == 0u;
            const unsigned leaders = __ballot_sync(0xffffffffu, leads);
            const int at = listed + __popc(leaders & ((1u << lane) - 1u));
            if (leads && at < LIST) {
              p.list_page[at] = page[n];
              p.list_index[at] = i;
              p.list_who[at] = same == everybody ? 0xffffffffu : same;
            }
            listed += __popc(leaders);
          }
          if (listed > LIST) listed = -1;
        }
        if (listed >= 0) total += listed;
      }
      if (listed < 0) {
        int base = shared_count;  // places in the list, tokens in order: lanes hold t, t + 32, ..
#pragma unroll
        for (int u = 0; u < EACH; ++u) {
          const int t = lane + 32 * u, first_own = max(common, low[u] / PAGE), own = max(0, pages[u] - first_own);
          int through = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            int other = __shfl_up_sync(0xffffffffu, through, o);
            if (lane >= o) through += other;
          }
          if (t < tokens) { p.list_index[t] = first_own; p.list_page[t] = base + through - own; }
          base += __shfl_sync(0xffffffffu, through, 31);
        }
        total = base;
      }
      if (lane == 0) {
        p.token0 = first + t0;
        p.tokens = tokens;
        p.row0 = row0;
        p.shared_first = least_first;
        p.shared_count = shared_count;
        p.total = total;
        p.listed = listed;
        p.longest = which;
        p.all_from = from;
        p.all_to = to;
      }
    }
  }
  __syncthreads();
}

// Who has a page: everybody (EVERYBODY), else a bit a token where the plan lists pages, else one token.
constexpr int EVERYBODY = -1;
__device__ __forceinline__ bool has_page(const Plan& p, int who, int token) {
  return who == EVERYBODY || (p.listed >= 0 ? ((unsigned)who >> (token & 31) & 1u) != 0u : who == token);
}
// Place i of the list: who has the page, and its index in the table rows.
__device__ __forceinline__ int look_up(const Plan& p, int i, int& who) {
  who = EVERYBODY;
  if (i < p.shared_count) return p.shared_first + i;
  if (p.listed >= 0) {
    who = (int)p.list_who[i - p.shared_count];
    return p.list_index[i - p.shared_count];
  }
  int lo = 0, hi = p.tokens - 1;  // the last token whose own pages begin at or before i
  while (lo < hi) {
    int mid = (lo + hi + 1) >> 1;
    if (p.list_page[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  who = lo;
  return p.list_index[lo] + i - p.list_page[lo];
}
__device__ __forceinline__ int page_at(const Plan& p, const Args& a, int i) {
  if (i >= p.shared_count && p.listed >= 0) return p.list_page[i - p.shared_count];
  int who, index = look_up(p, i, who);
  return a.cache.page_table[(size_t)p.slot[who == EVERYBODY ? p.longest : who] * a.cache.max_pages + index];
}

// A stretch of the list, at most LIST pages: page, first position, who has it.
struct Stretch { int page[LIST], at[LIST], who[LIST]; };
// (All threads call; ends with a barrier.)
__device__ __forceinline__ void fill(Stretch& l, const Plan& p, const Args& a, int begin, int end) {
  for (int i = begin + (int)threadIdx.x; i < end; i += blockDim.x) {
    l.at[i - begin] = look_up(p, i, l.who[i - begin]) * PAGE;
    l.page[i - begin] = page_at(p, a, i);
  }
  __syncthreads();
}

// ---- results: of a block, of a cluster, of all ------------------------------------------------------------------------
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n"
               "barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ unsigned remote_addr(const void* local, unsigned rank) {
  unsigned addr = (unsigned)__cvta_generic_to_shared(local), remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
__device__ __forceinline__ float2 remote_float2(unsigned addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 remote_float4(unsigned addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// (maximum, sum) of partial results together, the maxima as powers of two: what a part counts, and the sum. A sum beside a
// maximum of -inf is 0, or a NaN that has to stay one.
__device__ __forceinline__ float share_of(float m, float top) { return m > -INFINITY ? exp2f(m - top) : 0.f; }

template <typename T>
__device__ __forceinline__ void write_out(const Plan& p, const Args& a, int r, int d, float4 x, float sum) {
  const int per_kv = a.heads / a.cache.kv_heads, row = p.row0 + r, token = p.token0 + row / per_kv - p.row0 / per_kv;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  T* to = static_cast<T*>(a.out) + ((size_t)token * a.heads + blockIdx.y * per_kv + row % per_kv) * a.cache.head_dim + d;
  if (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(to) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
  } else {
    __nv_bfloat162 pair[2] = {__floats2bfloat162_rn(x.x * inv, x.y * inv), __floats2bfloat162_rn(x.z * inv, x.w * inv)};
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(pair);
  }
}

// Every block has its result in shared memory: x[row * ld ..] sums, ml[row] (maximum, sum); a block without pages has (-inf, 0)
// there and anything in x. The blocks of the cluster share the rows out, whole rows, so that whoever joins sums of a row also has
// written its maximum and sum (pieces dealt out in turn cross rows wherever a row's are no divisor of a block's threads). All
// threads call.
template <typename T, int ROWS>
__device__ __forceinline__ void finish(Plan& p, const Args& a, const float* x, int ld, const float2* ml) {
  const int hd = a.cache.head_dim, fours = hd / 4, clusters = a.splits / a.cluster;
  const unsigned size = a.cluster, rank = blockIdx.x % size;
  const int from = p.rows * rank / size * fours, to = p.rows * (rank + 1) / size * fours;  // this block's pieces
  const size_t pair = (size_t)blockIdx.z * gridDim.y + blockIdx.y;
  float* parts = a.scratch;
  float* part_ml = a.scratch + (size_t)gridDim.z * gridDim.y * clusters * ROWS * hd;
  if (size > 1) cluster_sync();
  else __syncthreads();
  for (int i = from + threadIdx.x; i < to; i += blockDim.x) {
    const int r = i / fours, d = (i % fours) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, total = 0.f;
    if (size == 1) {
      sum = *reinterpret_cast<const float4*>(x + r * ld + d);
      top = ml[r].x;
      total = ml[r].y;
      if (top == -INFINITY) sum = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      float2 each[MAX_CLUSTER];
      float4 v[MAX_CLUSTER];
#pragma unroll
      for (unsigned c = 0; c < MAX_CLUSTER; ++c)
        if (c < size) {
          each[c] = remote_float2(remote_addr(ml + r, c));
          v[c] = remote_float4(remote_addr(x + r * ld + d, c));
        }
#pragma unroll
      for (unsigned c = 0; c < MAX_CLUSTER; ++c)
        if (c < size) top = fmaxf(top, each[c].x);
#pragma unroll
      for (unsigned c = 0; c < MAX_CLUSTER; ++c)
        if (c < size) {
          const float w = share_of(each[c].x, top);
          total += each[c].x > -INFINITY ? w * each[c].y : each[c].y;
          if (w != 0.f) {
            sum.x = fmaf(w, v[c].x, sum.x); sum.y = fmaf(w, v[c].y, sum.y);
            sum.z = fmaf(w, v[c].z, sum.z); sum.w = fmaf(w, v[c].w, sum.w);
          }
        }
    }
    if (clusters == 1) {
      write_out<T>(p, a, r, d, sum, total);
    } else {
      const size_t at = (pair * clusters + blockIdx.x / size) * ROWS + r;
      *reinterpret_cast<float4*>(parts + at * hd + d) = sum;
      if (d == 0) *reinterpret_cast<float2*>(part_ml + at * 2) = make_float2(top, total);
    }
  }
  // Nobody leaves while others read its result. (With the order of memory: a value that a thread has asked for and does not use is
  // read too.)
  if (size > 1) cluster_sync();
  if (clusters == 1) return;
  // Blocks of one rank have written the same rows, one cluster's part each: the last of them joins these, in order.
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* ticket = a.tickets + pair * size + rank;
    unsigned before;  // (acquire and release: what the block has written, which the barrier has shown to this thread, and the others)
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(ticket) : "memory");
    p.last = before == (unsigned)(clusters - 1);
    if (p.last) *ticket = 0u;
  }
  __syncthreads();
  if (!p.last) return;
  for (int i = from + threadIdx.x; i < to; i += blockDim.x) {
    const int r = i / fours, d = (i % fours) * 4;
    float top = -INFINITY, total = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = 0; c0 < clusters; c0 += MAX_CLUSTER) {  // (eight parts at a time, the sum so far faded to the new maximum)
      float2 each[MAX_CLUSTER];
      float4 v[MAX_CLUSTER];
#pragma unroll
      for (int u = 0; u < MAX_CLUSTER; ++u)
        if (c0 + u < clusters) {
          const size_t at = (pair * clusters + c0 + u) * ROWS + r;
          each[u] = __ldcg(reinterpret_cast<const float2*>(part_ml + at * 2));
          v[u] = __ldcg(reinterpret_cast<const float4*>(parts + at * hd + d));
        }
      const float before = top;
#pragma unroll
      for (int u = 0; u < MAX_CLUSTER; ++u)
        if (c0 + u < clusters) top = fmaxf(top, each[u].x);
      const float fade = before > -INFINITY ? exp2f(before - top) : 1.f;
      total *= fade;
      sum.x *= fade; sum.y *= fade; sum.z *= fade; sum.w *= fade;
#pragma unroll
      for (int u = 0; u < MAX_CLUSTER; ++u)
        if (c0 + u < clusters) {
          const float w = share_of(each[u].x, top);
          total += each[u].x > -INFINITY ? w * each[u].y : each[u].y;
          if (w != 0.f) {
            sum.x = fmaf(w, v[u].x, sum.x); sum.y = fmaf(w, v[u].y, sum.y);
            sum.z = fmaf(w, v[u].z, sum.z); sum.w = fmaf(w, v[u].w, sum.w);
          }
        }
    }
    write_out<T>(p, a, r, d, sum, total);
  }
}

// ---- tensor cores ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void cp_async_16(void* smem, const void* gmem, bool valid) {
  unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  int bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(gmem), "r"(bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(unsigned* r, const void* p) {
  unsigned s = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldmatrix_x4_trans(unsigned* r, const void* p) {
  unsigned s = (unsigned)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void mma_bf16(float* c, const unsigned* a, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<unsigned*>(&v);
}
// Packed bfloat16: the sign bit's place of each that is not finite (an exponent of all ones carries into it); other bits mean
// nothing.
__device__ __forceinline__ unsigned odd_bits(unsigned v) { return (v & 0x7f807f80u) + 0x00800080u; }
__device__ __forceinline__ bool any_odd(unsigned bits) { return (bits & 0x80008000u) != 0u; }
// where piece `c` (16 bytes) of row r lies: neighbouring rows' pieces in different banks
template <int HD> __device__ __forceinline__ int place(int r, int c) {
  return r * HD + 8 * (HD >= 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3));
}

// Heads of 16, 32 and 48. Bound by the chain from the plan to the join: 9 heads on 3 of 32, 1 x 4 beams on 110 positions 7.2 us, 8 x 4
// on 1,020 10.7.
// HD: the head size, padded (32, 64). A warp has 16 * MT query rows; WM warps (of 4) lie one above another in the tile.
template <int HD, int MT, int WM, int STAGES>
__global__ void __launch_bounds__(WM * 128) mma_kernel(const Args a) {
  constexpr int THREADS = WM * 128, ROWS = 16 * MT * WM;
  constexpr bool KEEP_Q = MT * HD <= 128;  // the queries' operands stay in registers
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ Plan p;
  __shared__ Stretch list;
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  __shared__ float2 sm_ml[ROWS];
  bf16* q_s = reinterpret_cast<bf16*>(smem_raw);  // [ROWS][HD]
  bf16* ring = q_s + ROWS * HD;                    // per stage: keys [64][HD], values [64][HD]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int quarter = warp & 3, tier = warp >> 2;  // which 16 keys of a page; which of the tile's rows
  const int hd = a.cache.head_dim, pieces = hd >> 3, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  make_plan(p, a, ROWS);
  if (p.rows == 0) return;
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  float* sum = reinterpret_cast<float*>(ring);  // [4][ROWS][HD], at the end
  if (begin < end) {
    // queries (rows beyond the tile and dimensions beyond the head are zeros)
    const bf16* q = static_cast<const bf16*>(a.q);
    for (int i = tid; i < ROWS * (HD / 8); i += THREADS) {
      int r = i / (HD / 8), c = i % (HD / 8), row = p.row0 + r;
      bool ok = r < p.rows && c < pieces;
      const bf16* src = q;
      if (ok) src = q + ((size_t)(p.token0 + row / per_kv - p.row0 / per_kv) * a.heads + kv * per_kv + row % per_kv) * hd + c * 8;
      cp_async_16(q_s + place<HD>(r, c), src, ok);
    }
    if (pieces < HD / 8)
      for (int i = tid; i < STAGES * 2 * 64 * (HD / 8); i += THREADS) {
        int c = i % (HD / 8), r = i / (HD / 8);
        if (c >= pieces) *reinterpret_cast<uint4*>(ring + (size_t)(r >> 6) * 64 * HD + place<HD>(r & 63, c)) = make_uint4(0u, 0u, 0u, 0u);
      }
    cp_async_commit();
    // this thread's rows of the tile: 16 * MT * tier + 16 i + lane / 4 + 8 e
    int token[MT][2], high[MT][2], low[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int r = 16 * (MT * tier + i) + (lane >> 2) + 8 * e;
        bool real = r < p.rows;
        int t = real ? (p.row0 + r) / per_kv - p.row0 / per_kv : 0;
        token[i][e] = real ? t : -2;
        high[i][e] = real ? p.position[t] : -1;
        low[i][e] = real ? p.low[t] : 0;
      }
    float m[MT][2], l[MT][2], o[MT][HD / 8][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = 0.f;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
    }
    unsigned qf[KEEP_Q ? MT : 1][KEEP_Q ? HD / 16 : 1][4];
    const bf16* base = static_cast<const bf16*>(a.cache.base);
    const float scale = a.scale * 1.4426950408889634f;  // probabilities are powers of two

    for (int part = begin; part < end; part += LIST) {
      const int count = min(LIST, end - part);
      fill(list, p, a, part, part + count);
      auto bring = [&](int i) {
        bf16* keys = ring + (size_t)(i % STAGES) * 2 * 64 * HD;
        const int left = p.position[p.longest] - list.at[i];  // (rows that nobody sees are not read)
        const bf16* src = base + kv_offset(a.cache, list.page[i], 0, kv, 0);
        const size_t values = (size_t)a.cache.kv_heads * PAGE * hd;
        for (int c = tid; c < 64 * (HD / 8); c += THREADS) {
          int r = c / (HD / 8), d = c % (HD / 8);
          const bool ok = r <= left;
          if (d < pieces) {
            cp_async_16(keys + place<HD>(r, d), ok ? src + r * hd + d * 8 : base, ok);
            cp_async_16(keys + 64 * HD + place<HD>(r, d), ok ? src + values + r * hd + d * 8 : base, ok);
          }
        }
      };
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) {
        if (i < count) bring(i);
        cp_async_commit();
      }
      for (int it = 0; it < count; ++it) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();
        if (it + STAGES - 1 < count) bring(it + STAGES - 1);
        cp_async_commit();
        const bf16* keys = ring + (size_t)(it % STAGES) * 2 * 64 * HD;
        const bf16* vals = keys + 64 * HD;
        if (KEEP_Q && it == 0 && part == begin) {
#pragma unroll
          for (int i = 0; i < (KEEP_Q ? MT : 1); ++i)
#pragma unroll
            for (int k = 0; k < (KEEP_Q ? HD / 16 : 1); ++k)
              ldmatrix_x4(qf[i][k], q_s + place<HD>(16 * (MT * tier + i) + (lane & 15), 2 * k + (lane >> 4)));
        }
        const int who = list.who[it], at = list.at[it] + 16 * quarter;
        const bool whole = who == EVERYBODY && at >= p.all_from && at + 15 <= p.all_to;
        float s[MT][2][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][0][e] = s[i][1][e] = 0.f;
        // scores of 16 keys: keys as the second operand, dimensions in steps of 16
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          unsigned kf[4];
          ldmatrix_x4(kf, keys + place<HD>(16 * quarter + (lane & 7) + 8 * (lane >> 4), 2 * k + ((lane >> 3) & 1)));
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            unsigned q4[4];
            const unsigned* qa = qf[KEEP_Q ? i : 0][KEEP_Q ? k : 0];
            if (!KEEP_Q) {
              ldmatrix_x4(q4, q_s + place<HD>(16 * (MT * tier + i) + (lane & 15), 2 * k + (lane >> 4)));
              qa = q4;
            }
            mma_bf16(s[i][0], qa, kf[0], kf[1]);
            mma_bf16(s[i][1], qa, kf[2], kf[3]);
          }
        }
        unsigned seen[MT][2];  // of this thread's four keys of a row: which it sees
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = m[i][e];
            seen[i][e] = 15u;
            const bool mine = whole || (token[i][e] >= 0 && has_page(p, who, token[i][e]));
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                float v = s[i][j][2 * e + u] * scale;
                if (!whole) {
                  int key = at + 8 * j + 2 * (lane & 3) + u;
                  bool sees = mine && key <= high[i][e] && key >= low[i][e];
                  if (!sees) {
                    v = -INFINITY;
                    seen[i][e] &= ~(1u << (2 * j + u));
                  }
                }
                s[i][j][2 * e + u] = v;
                top = fmaxf(top, v);
              }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float shift = top > -INFINITY ? top : 0.f;
            if (top > m[i][e]) {
              const float fade = exp2f(m[i][e] - shift);
              m[i][e] = top;
              l[i][e] *= fade;
#pragma unroll
              for (int n = 0; n < HD / 8; ++n) {
                o[i][n][2 * e] *= fade;
                o[i][n][2 * e + 1] *= fade;
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                float w = fast_exp2(s[i][j][2 * e + u] - shift);
                s[i][j][2 * e + u] = w;
                l[i][e] += w;
              }
          }
        unsigned pf[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          pf[i][0] = pack_bf16(s[i][0][0], s[i][0][1]);
          pf[i][1] = pack_bf16(s[i][0][2], s[i][0][3]);
          pf[i][2] = pack_bf16(s[i][1][0], s[i][1][1]);
          pf[i][3] = pack_bf16(s[i][1][2], s[i][1][3]);
        }
        bool odd = false;
        if (!whole) {  // does a value that somebody may not see have to be kept out of the product?
          unsigned bits = 0u;
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            unsigned vf[4];
            ldmatrix_x4_trans(vf, vals + place<HD>(16 * quarter + (lane & 15), 2 * n + (lane >> 4)));
            bits |= odd_bits(vf[0]) | odd_bits(vf[1]) | odd_bits(vf[2]) | odd_bits(vf[3]);
          }
          odd = __any_sync(0xffffffffu, any_odd(bits));
        }
        if (!odd) {
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            unsigned vf[4];
            ldmatrix_x4_trans(vf, vals + place<HD>(16 * quarter + (lane & 15), 2 * n + (lane >> 4)));
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              mma_bf16(o[i][2 * n], pf[i], vf[0], vf[1]);
              mma_bf16(o[i][2 * n + 1], pf[i], vf[2], vf[3]);
            }
          }
        } else {
#pragma unroll
          for (int key = 0; key < 16; ++key) {
            const int holder = (lane & ~3) | ((key & 7) >> 1), bit = 2 * (key >> 3) + (key & 1);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float w = __shfl_sync(0xffffffffu, s[i][key >> 3][2 * e + (key & 1)], holder);
                unsigned sees = __shfl_sync(0xffffffffu, seen[i][e], holder) >> bit & 1u;
                w = __bfloat162float(__float2bfloat16_rn(w));
                if (sees) {
#pragma unroll
                  for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                      o[i][n][2 * e + u] = fmaf(w, __bfloat162float(vals[place<HD>(16 * quarter + key, n) + 2 * (lane & 3) + u]), o[i][n][2 * e + u]);
                }
              }
          }
        }
      }
      cp_async_wait<0>();
      __syncthreads();  // (the list and the ring are free again)
    }
    cp_async_wait<0>();
    // ---- the four quarters of a tier together: a common maximum, then sums through shared memory
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (high[i][e] < 0) { m[i][e] = -INFINITY; l[i][e] = 0.f; }  // (a row that sees nothing)
        l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 1);
        l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 2);
        int r = 16 * (MT * tier + i) + (lane >> 2) + 8 * e;
        if ((lane & 3) == 0) { sm_m[quarter][r] = m[i][e]; sm_l[quarter][r] = l[i][e]; }
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int r = 16 * (MT * tier + i) + (lane >> 2) + 8 * e;
        float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
        float w = share_of(m[i][e], top);
        // (rows without a key in this quarter: nothing, whatever the products made of zeros)
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          float2 v = make_float2(0.f, 0.f);
          if (w != 0.f) v = make_float2(o[i][n][2 * e] * w, o[i][n][2 * e + 1] * w);
          *reinterpret_cast<float2*>(sum + ((size_t)quarter * ROWS + r) * HD + 8 * n + 2 * (lane & 3)) = v;
        }
      }
    __syncthreads();
    for (int i = tid; i < ROWS * (HD / 4); i += THREADS) {  // (into the first quarter's place)
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float4 x = *reinterpret_cast<const float4*>(sum + ((size_t)w * ROWS + r) * HD + d);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      *reinterpret_cast<float4*>(sum + (size_t)r * HD + d) = v;
      if (d == 0) {
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, sm_m[w][r]);
#pragma unroll
        for (int w = 0; w < 4; ++w) total += sm_m[w][r] > -INFINITY ? sm_l[w][r] * exp2f(sm_m[w][r] - top) : sm_l[w][r];
        sm_ml[r] = make_float2(top, total);
      }
    }
  } else {
    for (int r = tid; r < ROWS; r += THREADS) sm_ml[r] = make_float2(-INFINITY, 0.f);
  }
  finish<bf16, ROWS>(p, a, sum, HD, sm_ml);
}

template <typename Kernel, typename... Rest>
int launch_clusters(Kernel kernel, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream, const Rest&... rest) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  int n = 0;
  if (cluster > 1) {
    attributes[n].id = cudaLaunchAttributeClusterDimension;
    attributes[n].val.clusterDim.x = cluster;
    attributes[n].val.clusterDim.y = 1;
    attributes[n++].val.clusterDim.z = 1;
  }
  if (dllm_pdl_enabled()) {
    attributes[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  config.attrs = attributes;
  config.numAttrs = n;
  return cudaLaunchKernelEx(&config, kernel, rest...) == cudaSuccess ? DLLM_OK : DLLM_LAUNCH_FAILED;
}

// ---- 5th-generation tensor cores -----------------------------------------------------------------------------------
// A step takes two pages, 128 keys. The query rows are few, so keys and values are the operands of 128 rows and the query
// rows the columns of both products: S^T = K Q^T (keys x rows), O^T += V^T P^T (dimensions x rows; keys and values as they lie in
// their pages, P^T written as [key][row]). A product then reads 128 x 16 values of a page and ROWS x 16 others; with the query
// rows as the 128-row operand (padded) it would read those 128 x 16 for every 64 keys: 768 cycles of shared memory a page
// for heads of 128 instead of 320.
//   softmax warps  GROUPS groups that take the steps in turn, each with scores, P and outputs of its own: a thread has a key
//                  and 32 query rows. A row's maximum over the step goes through redux and shared memory; where it grew the
//                  group's outputs are scaled in tensor memory (32 columns). Every step uses the running maximum itself, so
//                  that the largest weight is 1 and not rounded. Three groups for heads of 64, two above, one for two blocks of a
//                  multiprocessor, and one where there are 64 rows: a second left 96 registers a thread and 200 bytes
//                  spilled (9 heads on 3 of 64, 16 new tokens on 1,000 positions 10.9 us, 9.0 with one; 32 on 8 of 128, eight
//                  prompts of 16,000, 117.8 and 109.3; 8 x 16 beams on 2,000 37.9 and 39.3).
//   three more     one looks pages up, 32 at a time, and issues their TMA loads; one issues the scores' products, one the
//                  outputs'.
// Pages that some row sees in part are looked at: a value that is not finite is kept out of the product; such a step is added
// by the softmax warps, key by key.
// Every wait is bounded; a role that gives up sets the status word and leaves.
// Bound by HBM where pages are many: two chunks of eight tokens on 40,000 positions, 32 heads on 8 of 128, 56.3 us (287 MB, 5.1 TB/s, 128
// blocks); by the chain lookup, page, scores, softmax, outputs, join where they are few: 8 x 8 beams on 2,150 positions 26.3 us (77 MB,
// two blocks a pair of prompt and kv head), 1 x 4 on 110, 9 heads on 3 of 64, 8.8 us, of which 2 are the plan, 2 the first page, 3 the join.
namespace t5 {
using namespace tc5;
constexpr int KEYS = 2 * PAGE;
constexpr int P_BYTES = KEYS * 128;  // [key][64 rows]

template <int BOXES, int ROWS, int GROUPS> struct Shape {
  static constexpr int BLOCKS = GROUPS == 1 && ROWS == 32 ? 2 : 1;  // of a multiprocessor
  static constexpr int HALVES = ROWS / 32;                      // warps that share a step's keys, 32 rows each
  static constexpr int GROUP = 4 * HALVES, SOFT_WARPS = GROUPS * GROUP, THREADS = (SOFT_WARPS + 3) * 32;
  static constexpr int K_STAGES = BOXES == 2 || BLOCKS == 2 ? 2 : 4, V_STAGES = BLOCKS == 2 ? 2 : BOXES == 2 ? 3 : 5;
  static constexpr int Q_BYTES = BOXES * ROWS * 128, KV_BYTES = BOXES * KEYS * 128;
  static constexpr unsigned COLUMNS = 2 * GROUPS * ROWS > 128 ? 256 : 2 * GROUPS * ROWS > 64 ? 128 : 64;  // of tensor memory: scores and outputs
  static constexpr int SMEM = Q_BYTES + GROUPS * P_BYTES + (K_STAGES + V_STAGES) * KV_BYTES + 1024;
  static constexpr int LD = BOXES * 64 + 4;  // floats of a row of the results at the end, which lie in the stages' place
  static_assert(GROUPS * ROWS * LD * 4 <= (K_STAGES + V_STAGES) * KV_BYTES, "results");
};

struct Barriers {
  uint64_t k_full[4], k_empty[4], v_full[5], v_empty[5], s_full[4], s_empty[4], p_full[4], o_full[4];
};

// An operand whose rows of 128 bytes (64 values of M or N) are its K index; `next`: bytes from 64 values of M or N to the next.
__device__ __forceinline__ uint64_t transposed_desc(unsigned addr, unsigned next) {
  return (smem_desc(addr) & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(next >> 4) << 16);
}
__device__ __forceinline__ float largest_of_warp(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// two floats at a time
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 apart(Two v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int BOXES, int ROWS, int GROUPS>
__global__ void __launch_bounds__(Shape<BOXES, ROWS, GROUPS>::THREADS, Shape<BOXES, ROWS, GROUPS>::BLOCKS)
    kernel(const __grid_constant__ CUtensorMap map_kv, const Args a) {
  typedef Shape<BOXES, ROWS, GROUPS> S;
  constexpr int K_STAGES = S::K_STAGES, V_STAGES = S::V_STAGES, KV_BYTES = S::KV_BYTES, SOFT_WARPS = S::SOFT_WARPS;
  constexpr int BOX = KEYS * 128;  // bytes of 64 columns of a step's keys or values
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // swizzle atoms: 1 KB
  unsigned char* q_s = tiles;
  unsigned char* p_s = q_s + S::Q_BYTES;
  unsigned char* k_s = p_s + GROUPS * P_BYTES;
  unsigned char* v_s = k_s + K_STAGES * KV_BYTES;
  __shared__ Plan p;
  __shared__ Barriers bar;
  __shared__ unsigned tmem_base_s;
  __shared__ __align__(16) float sm_max[2][GROUPS][4][ROWS];    // a step's maxima, by the warp of 32 keys (two sets, in turn)
  __shared__ __align__(16) float sm_shift[SOFT_WARPS][32], sm_fade[SOFT_WARPS][32];
  __shared__ float sm_m[GROUPS][ROWS], sm_l[GROUPS][4][ROWS];
  __shared__ float2 sm_ml[ROWS];
  __shared__ int odd_s[GROUPS], skip_s[GROUPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = a.cache.head_dim, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads;
  if (tid == 0) {
    for (int s = 0; s < K_STAGES; ++s) { mbar_init(&bar.k_full[s], 1); mbar_init(&bar.k_empty[s], 1); }
    for (int s = 0; s < V_STAGES; ++s) { mbar_init(&bar.v_full[s], 1); mbar_init(&bar.v_empty[s], 1); }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.s_empty[i], S::GROUP);
      mbar_init(&bar.p_full[i], S::GROUP);
      mbar_init(&bar.o_full[i], 1);
      odd_s[i] = skip_s[i] = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
  }
  // (tensor memory is this block's before the next kernel's blocks may come and ask for theirs)
  if (warp == SOFT_WARPS + 1) tmem_alloc(&tmem_base_s, S::COLUMNS);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  pdl_launch_dependents();
  pdl_wait();
  if (warp >= 1 && warp < SOFT_WARPS) {  // (beside the first warp, which makes the plan)
    // the queries: rows beyond the tile and dimensions beyond the head are zeros; they carry the scale's sign, or that it is 0
    const int first = a.cuts[blockIdx.z / a.tiles], row0 = (int)(blockIdx.z % a.tiles) * ROWS;
    const int rows = (a.cuts[blockIdx.z / a.tiles + 1] - first) * per_kv - row0;
    const bf16* q = static_cast<const bf16*>(a.q);
    for (int i = tid - 32; i < ROWS * BOXES * 8; i += SOFT_WARPS * 32 - 32) {
      const int r = i / (BOXES * 8), c = i % (BOXES * 8), row = row0 + r;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && c * 8 < hd)
        v = *reinterpret_cast<const uint4*>(q + ((size_t)(first + row / per_kv) * a.heads + kv * per_kv + row % per_kv) * hd + c * 8);
      if (a.scale == 0.f) v = make_uint4(0u, 0u, 0u, 0u);
      if (a.scale < 0.f) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
      *reinterpret_cast<uint4*>(q_s + (c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  make_plan(p, a, ROWS);
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  const int pages = p.rows ? end - begin : 0, steps = (pages + 1) / 2;
  float* ex = reinterpret_cast<float*>(k_s);  // at the end: results [GROUPS][ROWS][LD]
  if (steps > 0) {
    const unsigned tmem_s = tmem_base_s, tmem_o = tmem_base_s + GROUPS * ROWS;
    if (warp == SOFT_WARPS) {
      int issued_k = 0, issued_v = 0;
      bool ok = true;
      for (int j0 = 0; j0 < steps && ok; j0 += 16) {
        const int page = 2 * j0 + lane < pages ? page_at(p, a, begin + 2 * j0 + lane) : 0;
        for (int u = 0; u < 16 && j0 + u < steps && ok; ++u) {
          const int j = j0 + u, sk = j % K_STAGES, sv = j % V_STAGES, count = min(2, pages - 2 * j);
          const int at[2] = {__shfl_sync(0xffffffffu, page, 2 * u), __shfl_sync(0xffffffffu, page, 2 * u + 1)};
          if (lane == 0) {
            if (j >= K_STAGES && !mbar_wait(&bar.k_empty[sk], (j / K_STAGES - 1) & 1)) ok = false;
            if (ok) {
              mbar_expect_tx(&bar.k_full[sk], count * (KV_BYTES / 2));
              for (int c = 0; c < count; ++c)
#pragma unroll
                for (int x = 0; x < BOXES; ++x)
                  tma_load_2d(k_s + sk * KV_BYTES + x * BOX + c * (PAGE * 128), &map_kv, &bar.k_full[sk], x * 64,
                              ((at[c] * 2 + 0) * a.cache.kv_heads + kv) * PAGE);
              issued_k = j + 1;
              if (j >= V_STAGES && !mbar_wait(&bar.v_empty[sv], (j / V_STAGES - 1) & 1)) ok = false;
            }
            if (ok) {
              mbar_expect_tx(&bar.v_full[sv], count * (KV_BYTES / 2));
              for (int c = 0; c < count; ++c)
#pragma unroll
                for (int x = 0; x < BOXES; ++x)
                  tma_load_2d(v_s + sv * KV_BYTES + x * BOX + c * (PAGE * 128), &map_kv, &bar.v_full[sv], x * 64,
                              ((at[c] * 2 + 1) * a.cache.kv_heads + kv) * PAGE);
              issued_v = j + 1;
            }
          }
          ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        }
      }
      if (!ok && lane == 0) {  // gave up: nothing may land in this block's shared memory after it has left
        *(volatile int*)a.status = 52;
        for (int j = max(0, issued_k - K_STAGES); j < issued_k; ++j) mbar_wait(&bar.k_full[j % K_STAGES], (j / K_STAGES) & 1);
        for (int j = max(0, issued_v - V_STAGES); j < issued_v; ++j) mbar_wait(&bar.v_full[j % V_STAGES], (j / V_STAGES) & 1);
      }
    } else if (warp == SOFT_WARPS + 1) {
      if (lane == 0) {
        constexpr unsigned idesc = instr_desc(128, ROWS);
        const uint64_t q_desc = smem_desc(smem_u32(q_s));
        bool ok = true;
        for (int i = 0; i < steps && ok; ++i) {  // (a single last page: the other 64 rows are whatever lies there, and nobody looks)
          const int g = i % GROUPS, s = i % K_STAGES;
          ok = mbar_wait(&bar.k_full[s], (i / K_STAGES) & 1) && (i < GROUPS || mbar_wait(&bar.s_empty[g], (i / GROUPS - 1) & 1));
          if (!ok) break;
          fence_after_sync();
          const uint64_t k_desc = smem_desc(smem_u32(k_s + s * KV_BYTES));  // (start addresses / 16 are the low bits)
#pragma unroll
          for (int k = 0; k < BOXES * 4; ++k)
            if (k * 16 < hd)
              umma(tmem_s + (unsigned)(g * ROWS), k_desc + (((k >> 2) * BOX + (k & 3) * 32) >> 4),
                   q_desc + (((k >> 2) * (ROWS * 128) + (k & 3) * 32) >> 4), idesc, k > 0 ? 1u : 0u);
          tcgen05_commit(&bar.k_empty[s]);
          tcgen05_commit(&bar.s_full[g]);
        }
        if (!ok) *(volatile int*)a.status = 53;
      }
    } else if (warp == SOFT_WARPS + 2) {
      if (lane == 0) {
        constexpr unsigned idesc = instr_desc(128, ROWS, true) | (1u << 15);  // both operands' rows are keys
        for (int i = 0; i < steps; ++i) {
          const int g = i % GROUPS, s = i % V_STAGES;
          if (!mbar_wait(&bar.p_full[g], (i / GROUPS) & 1) || !mbar_wait(&bar.v_full[s], (i / V_STAGES) & 1)) {
            *(volatile int*)a.status = 54;
            break;
          }
          fence_after_sync();
          if (!*(volatile int*)&skip_s[g]) {
            // (heads of 64: the lower half of the 128 rows comes twice)
            const uint64_t v_desc = transposed_desc(smem_u32(v_s + s * KV_BYTES), BOXES == 2 ? BOX : 0);
            const uint64_t p_desc = smem_desc(smem_u32(p_s + g * P_BYTES));
            const int sixteens = min(8, 4 * (pages - 2 * i));
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < sixteens)
                umma(tmem_o + (unsigned)(g * ROWS), v_desc + ((k * 2048) >> 4), p_desc + ((k * 2048) >> 4), idesc,
                     (k > 0 || i >= GROUPS) ? 1u : 0u);
          }
          tcgen05_commit(&bar.v_empty[s]);
          tcgen05_commit(&bar.o_full[g]);
        }
      }
    } else {
      const int g = warp / S::GROUP, half = (warp % S::GROUP) >> 2, quarter = warp & 3;  // 32 keys of the step; 32 of the rows
      const int key = quarter * 32 + lane, row0 = half * 32, in_group = tid - g * S::GROUP * 32;
      const unsigned lanes = (unsigned)(quarter * 32) << 16;
      const unsigned s_addr = tmem_s + lanes + (unsigned)(g * ROWS + row0), o_addr = tmem_o + lanes + (unsigned)(g * ROWS + row0);
      unsigned char* p_row = p_s + g * P_BYTES + key * 128;
      // this lane's row of the 32 (every warp of the half keeps the same)
      const int row = row0 + lane;
      const bool real = row < p.rows;
      const int token = real ? (p.row0 + row) / per_kv - p.row0 / per_kv : 0;
      const int high = real ? p.position[token] : -1, low = real ? p.low[token] : 0;
      // (the queries carry the sign: the largest product is the largest score; and a masked product is -inf, which 0 must not meet)
      const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f;
      const Two scale2 = two(scale, scale);
      float m_run = -INFINITY;  // of this lane's row
      Two l[16];                // of all 32 rows, this thread's keys
#pragma unroll
      for (int c = 0; c < 16; ++c) l[c] = two(0.f, 0.f);
      bool ok = true;
      int taken = 0;
      // (a wait that ran out is not left at once: the warps of a group meet at barriers that they all have to reach)
      for (int j = g; j < steps; j += GROUPS, ++taken) {
        int who0, who1 = EVERYBODY;
        const int at0 = look_up(p, begin + 2 * j, who0) * PAGE;
        const bool second = 2 * j + 1 < pages;
        const int at1 = second ? look_up(p, begin + 2 * j + 1, who1) * PAGE : 0;
        const bool edge0 = who0 != EVERYBODY || at0 < p.all_from || at0 + PAGE - 1 > p.all_to;
        const bool edge1 = second && (who1 != EVERYBODY || at1 < p.all_from || at1 + PAGE - 1 > p.all_to);
        const bool upper = quarter >= 2;  // this warp's page of the two
        const int position0 = (upper ? at1 : at0) + (quarter & 1) * 32, who = upper ? who1 : who0;  // (of the warp's first key)
        const bool edge = upper ? edge1 : edge0, none = upper && !second;
        ok = ok && mbar_wait(&bar.s_full[g], (j / GROUPS) & 1);
        __syncwarp();
        fence_after_sync();
        float s[32];
        tmem_load16_nowait(s_addr, reinterpret_cast<unsigned*>(s));
        tmem_load16_nowait(s_addr + 16u, reinterpret_cast<unsigned*>(s) + 16);
        tmem_wait_ld();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.s_empty[g]);
        unsigned seen = none ? 0u : 0xffffffffu;  // rows that see this thread's key
        if (edge) {
          // a lane's row sees these of the warp's 32 keys; turned round, a lane's key is seen by these of the 32 rows
          const int last = high - position0, first = low - position0;
          seen = real && last >= 0 && first < 32 && has_page(p, who, token) ? 0xffffffffu : 0u;
          if (last < 31) seen &= 0xffffffffu >> (31 - max(last, 0));
          if (first > 0) seen &= 0xffffffffu << (first & 31);
          unsigned low_half = 0x0000ffffu;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const unsigned other = __shfl_xor_sync(0xffffffffu, seen, o);
            seen = lane & o ? (seen & ~low_half) | (other >> o & low_half) : (seen & low_half) | ((other & low_half) << o);
            low_half ^= low_half << (o >> 1);
          }
        }
        if (edge || none) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (!(seen >> c & 1u)) s[c] = -INFINITY;
        }
        // the rows' maxima over the step
        float* maxima = &sm_max[taken & 1][g][0][row0];
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 top = make_float4(largest_of_warp(s[c]), largest_of_warp(s[c + 1]), largest_of_warp(s[c + 2]), largest_of_warp(s[c + 3]));
          if (lane == 0) *reinterpret_cast<float4*>(&maxima[quarter * ROWS + c]) = top;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(2 + g * S::HALVES + half) : "memory");
        const float largest = fmaxf(fmaxf(maxima[lane], maxima[ROWS + lane]), fmaxf(maxima[2 * ROWS + lane], maxima[3 * ROWS + lane]));
        const float top = largest * scale;
        float fade = 1.f;
        if (top > m_run) {
          if (m_run > -INFINITY) fade = fast_exp2(m_run - top);  // (else the row's outputs are zeros so far)
          m_run = top;
        }
        const bool fades = __any_sync(0xffffffffu, fade != 1.f);
        sm_shift[warp][lane] = m_run > -INFINITY ? -m_run : 0.f;
        if (fades) sm_fade[warp][lane] = fade;
        __syncwarp();
        if (fades) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            asm volatile("" ::: "memory");  // (what comes next is not fetched ahead: registers)
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sm_fade[warp][c]);
            l[c / 2] = mul2(l[c / 2], f.x);
            l[c / 2 + 1] = mul2(l[c / 2 + 1], f.y);
          }
        }
        // the group's previous product has to be over: it reads P and adds to the outputs
        if (taken >= 1) {
          ok = ok && mbar_wait(&bar.o_full[g], (taken - 1) & 1);
          __syncwarp();
          fence_after_sync();
        }
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          asm volatile("" ::: "memory");
          unsigned packed[4];
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const ulonglong2 shift = *reinterpret_cast<const ulonglong2*>(&sm_shift[warp][c + e]);
            const float2 x = apart(fma2(two(s[c + e], s[c + e + 1]), scale2, shift.x));
            const float2 y = apart(fma2(two(s[c + e + 2], s[c + e + 3]), scale2, shift.y));
            const float w0 = fast_exp2(x.x), w1 = fast_exp2(x.y), w2 = fast_exp2(y.x), w3 = fast_exp2(y.y);
            packed[e / 2] = pack_bf16(w0, w1);
            packed[e / 2 + 1] = pack_bf16(w2, w3);
            l[(c + e) / 2] = add2(l[(c + e) / 2], two(w0, w1));
            l[(c + e) / 2 + 1] = add2(l[(c + e) / 2 + 1], two(w2, w3));
          }
          *reinterpret_cast<uint4*>(p_row + (((half * 4 + c / 8) ^ (key & 7)) << 4)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
        bool odd = false;
        const unsigned char* v_tile = v_s + (j % V_STAGES) * KV_BYTES;
        if (edge0 || edge1) {
          ok = ok && mbar_wait(&bar.v_full[j % V_STAGES], (j / V_STAGES) & 1);
          unsigned bits = 0u;
#pragma unroll
          for (int x = 0; x < BOXES; ++x)
#pragma unroll
            for (int i = 0; i < BOX / 16 / (S::GROUP * 32); ++i) {
              const int at = (i * S::GROUP * 32 + in_group) * 16;
              if (second || at < PAGE * 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(v_tile + x * BOX + at);
                bits |= odd_bits(v.x) | odd_bits(v.y) | odd_bits(v.z) | odd_bits(v.w);
              }
            }
          if (__any_sync(0xffffffffu, any_odd(bits)) && lane == 0) odd_s[g] = 1;
          asm volatile("bar.sync %0, %1;" ::"r"(6 + g), "n"(S::GROUP * 32) : "memory");
          odd = *(volatile int*)&odd_s[g] != 0;
          asm volatile("bar.sync %0, %1;" ::"r"(6 + g), "n"(S::GROUP * 32) : "memory");
          if (in_group == 0) { odd_s[g] = 0; *(volatile int*)&skip_s[g] = odd; }
        } else if (in_group == 0) {
          *(volatile int*)&skip_s[g] = 0;
        }
        if (odd || (taken >= 1 && fades)) {
#pragma unroll
          for (int c0 = 0; c0 < 32; c0 += 16) {
            unsigned o[16];  // of this thread's dimension, 16 of the rows
            if (taken >= 1) tmem_load16(o_addr + (unsigned)c0, o);
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              asm volatile("" ::: "memory");
              if (taken == 0) o[c] = o[c + 1] = o[c + 2] = o[c + 3] = 0u;
              if (fades) {
                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sm_fade[warp][c0 + c]);
                const float2 x = apart(mul2(two(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), f.x));
                const float2 y = apart(mul2(two(__uint_as_float(o[c + 2]), __uint_as_float(o[c + 3])), f.y));
                o[c] = __float_as_uint(x.x); o[c + 1] = __float_as_uint(x.y);
                o[c + 2] = __float_as_uint(y.x); o[c + 3] = __float_as_uint(y.y);
              }
            }
            if (odd) {
              const int d = quarter * 32 + lane, keys = second ? KEYS : PAGE;  // (heads of 64: dimensions beyond are not used)
#pragma unroll 1
              for (int k = 0; k < keys; ++k) {
                const int at_k = (k < PAGE ? at0 : at1) + (k & (PAGE - 1));
                const unsigned have = __ballot_sync(0xffffffffu, real && has_page(p, k < PAGE ? who0 : who1, token) && at_k <= high && at_k >= low);
                const float x = __bfloat162float(*reinterpret_cast<const bf16*>(
                    v_tile + (BOXES == 2 ? d >> 6 : 0) * BOX + k * 128 + ((((d & 63) >> 3) ^ (k & 7)) << 4) + 2 * (d & 7)));
                const unsigned char* weights = p_s + g * P_BYTES + k * 128;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                  const int r = row0 + c0 + c;
                  const float w = __bfloat162float(*reinterpret_cast<const bf16*>(weights + (((r >> 3) ^ (k & 7)) << 4) + 2 * (r & 7)));
                  if (have >> (c0 + c) & 1u) o[c] = __float_as_uint(fmaf(w, x, __uint_as_float(o[c])));
                }
              }
            }
            tmem_store16(o_addr + (unsigned)c0, o);
          }
          tmem_wait_st();
          fence_before_sync();
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.p_full[g]);
      }
      if (ok && taken >= 1) ok = mbar_wait(&bar.o_full[g], (taken - 1) & 1);
      if (!ok) *(volatile int*)a.status = 55;
      __syncwarp();
      fence_after_sync();
      // ---- the groups together. Lane c ends with row c's sum over the warp's 32 keys: pairs of lanes share their rows out, then fours, ..
      float sums[32];
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float2 x = apart(l[c]);
        sums[2 * c] = x.x;
        sums[2 * c + 1] = x.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int c = 0; c < o; ++c) {
          const float give = up ? sums[c] : sums[c + o], keep = up ? sums[c + o] : sums[c];
          sums[c] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
      }
      if (high < 0) m_run = -INFINITY;  // (a row that sees nothing)
      sm_l[g][quarter][row] = high < 0 ? 0.f : sums[0];
      if (quarter == 0) sm_m[g][row] = m_run;
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      float most = sm_m[0][row];
#pragma unroll
      for (int i = 1; i < GROUPS; ++i) most = fmaxf(most, sm_m[i][row]);
      const float w = share_of(m_run, most);
      const int d = quarter * 32 + lane, active = min(GROUPS, steps);  // (groups that have had a step)
      if (taken >= 1) {
#pragma unroll
        for (int c0 = 0; c0 < 32; c0 += 16) {
          unsigned o[16];
          tmem_load16(o_addr + (unsigned)c0, o);
          float* to = ex + (size_t)(g * ROWS + row0 + c0) * S::LD + d;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float wc = __shfl_sync(0xffffffffu, w, c0 + c);
            if (d < BOXES * 64) to[c * S::LD] = wc != 0.f ? __uint_as_float(o[c]) * wc : 0.f;
          }
        }
      }
      if (g == 0 && quarter == 0) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
          const float part = (sm_l[i][0][row] + sm_l[i][1][row]) + (sm_l[i][2][row] + sm_l[i][3][row]);
          total += sm_m[i][row] > -INFINITY ? part * share_of(sm_m[i][row], most) : part;
        }
        sm_ml[row] = make_float2(most, total);
      }
      if (active > 1) asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      for (int i = active > 1 ? tid : ROWS * (BOXES * 16); i < ROWS * (BOXES * 16); i += SOFT_WARPS * 32) {  // (into the first group's place)
        float4* x = reinterpret_cast<float4*>(ex + (size_t)(i / (BOXES * 16)) * S::LD + (i % (BOXES * 16)) * 4);
        float4 z = *x;
#pragma unroll
        for (int e = 1; e < GROUPS; ++e) {
          if (e >= active) break;
          const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + (size_t)e * ROWS * S::LD);
          z.x += y.x; z.y += y.y; z.z += y.z; z.w += y.w;
        }
        *x = z;
      }
    }
    fence_before_sync();
  } else {
    for (int r = tid; r < ROWS; r += S::THREADS) sm_ml[r] = make_float2(-INFINITY, 0.f);
  }
  __syncthreads();
  if (warp == SOFT_WARPS + 1) tmem_dealloc(tmem_base_s, S::COLUMNS);
  if (p.rows == 0) return;
  finish<bf16, ROWS>(p, a, ex, S::LD, sm_ml);
}

template <int BOXES, int ROWS, int GROUPS>
int launch(const Args& a, long long pages, dim3 grid, cudaStream_t stream) {
  typedef Shape<BOXES, ROWS, GROUPS> S;
  CUtensorMap map;
  if (!make_map(&map, a.cache.base, pages * 2 * a.cache.kv_heads * PAGE, a.cache.head_dim, PAGE)) return DLLM_LAUNCH_FAILED;
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)kernel<BOXES, ROWS, GROUPS>, S::SMEM, done)) return DLLM_LAUNCH_FAILED;
  return launch_clusters(kernel<BOXES, ROWS, GROUPS>, grid, S::THREADS, S::SMEM, a.cluster, stream, map, a);
}
}  // namespace t5

// ---- everything else ---------------------------------------------------------------------------------------------
// 16 query rows a tile, 256 threads, pages by cp.async into a ring of one or two stages, in the cache's type. Scores: a thread has one of
// a page's 64 keys and four rows. The rows' maxima go through shared memory, the weights of a key's 16 rows lie side by side in
// it. Sums: a thread has four dimensions and four rows, and every n-th key; the n groups are added at the end.
// Bound by a page's chain (scores 1.0 us, maxima 0.4, weights 0.3, sums 0.9 for heads of 64 in float32: shared-memory reads and their
// latency with eight warps): 9 heads on 3 of 64, 2 x 5 beams on 770 positions 14.2 us, 8 x 8 on 1,070 30. Half the instructions did
// not shorten it (packed multiply-adds, four keys a thread with the dimensions over four lanes, redux: 17.1 us where it was 17.0).
constexpr int FMA_ROWS = 16, FMA_THREADS = 256, FMA_DIM = 256, FMA_LD = 20;
constexpr int FMA_MOST = 152 << 10;  // bytes of dynamic shared memory: heads of 128 in float32, two stages; of 256, one

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four(const bf16* p) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <typename T> __host__ __device__ constexpr int fma_row(int hd) { return hd + 16 / (int)sizeof(T); }  // a page's row in shared memory
template <typename T> __host__ __device__ constexpr int fma_stages(int hd) { return hd * (int)sizeof(T) <= 512 ? 2 : 1; }

template <typename T>
__global__ void __launch_bounds__(FMA_THREADS) fma_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ Plan p;
  __shared__ Stretch list;
  __shared__ __align__(16) float sm_p[PAGE * FMA_LD];
  __shared__ float sm_max[2][2][FMA_ROWS], sm_l[2][FMA_ROWS];
  __shared__ __align__(16) float sm_fade[FMA_ROWS];  // (read by fours)
  __shared__ float2 sm_ml[FMA_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = a.cache.head_dim, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads;
  const int ld = hd + 4, row = fma_row<T>(hd), stages = fma_stages<T>(hd), fours = hd / 4;
  float* q_s = reinterpret_cast<float*>(smem_raw);             // [FMA_ROWS][ld]; at the end the sums
  T* ring = reinterpret_cast<T*>(q_s + FMA_ROWS * ld);         // per stage: keys, values [PAGE][row]
  float* groups_s = q_s + FMA_ROWS * ld;                       // at the end: [groups][FMA_ROWS][ld]
  pdl_launch_dependents();
  pdl_wait();
  if (warp >= 1) {  // (beside the first warp, which makes the plan)
    const int first = a.cuts[blockIdx.z / a.tiles], row0 = (int)(blockIdx.z % a.tiles) * FMA_ROWS;
    const int rows = (a.cuts[blockIdx.z / a.tiles + 1] - first) * per_kv - row0;
    for (int i = tid - 32; i < FMA_ROWS * fours; i += FMA_THREADS - 32) {
      const int r = i / fours, d = (i % fours) * 4, at = row0 + r;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) v = four(static_cast<const T*>(a.q) + ((size_t)(first + at / per_kv) * a.heads + kv * per_kv + at % per_kv) * hd + d);
      *reinterpret_cast<float4*>(q_s + r * ld + d) = v;
    }
  }
  make_plan(p, a, FMA_ROWS);
  if (p.rows == 0) return;
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  if (begin < end) {
    const T* base = static_cast<const T*>(a.cache.base);
    const float scale = a.scale * 1.4426950408889634f;
    // scores: this thread's key and rows
    const int key = (warp >> 2) * 32 + lane, r0 = (warp & 3) * 4;
    int token[4], high[4], low[4];
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool real = r0 + i < p.rows;
      token[i] = real ? (p.row0 + r0 + i) / per_kv - p.row0 / per_kv : -1;
      high[i] = real ? p.position[token[i]] : -1;
      low[i] = real ? p.low[token[i]] : 0;
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
    // sums: this thread's dimensions, rows and keys
    const int each = fours * 4, n_groups = min(16, FMA_THREADS / each), group = tid / each;
    const int d4 = (tid % each) % fours * 4, s0 = (tid % each) / fours * 4;
    float4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int chunks = hd * (int)sizeof(T) / 16;
    for (int part = begin; part < end; part += LIST) {
      const int count = min(LIST, end - part);
      fill(list, p, a, part, part + count);
      auto bring = [&](int i) {
        const T* keys = base + kv_offset(a.cache, list.page[i], 0, kv, 0);
        const size_t values = (size_t)a.cache.kv_heads * PAGE * hd;
        T* to = ring + (size_t)(i % stages) * 2 * PAGE * row;
        for (int c = tid; c < PAGE * chunks; c += FMA_THREADS) {
          const int r = c / chunks, d = c % chunks * (16 / (int)sizeof(T));
          cp_async_16(to + r * row + d, keys + r * hd + d, true);
          cp_async_16(to + (PAGE + r) * row + d, keys + values + r * hd + d, true);
        }
      };
      bring(0);
      cp_async_commit();
      for (int it = 0; it < count; ++it) {
        if (stages > 1) {
          if (it + 1 < count) bring(it + 1);
          cp_async_commit();
          cp_async_wait<1>();
        } else {
          cp_async_wait<0>();
        }
        __syncthreads();
        const T* keys = ring + (size_t)(it % stages) * 2 * PAGE * row;
        const T* vals = keys + PAGE * row;
        const int who = list.who[it], at = list.at[it];
        float s[4] = {0.f, 0.f, 0.f, 0.f};
        for (int d = 0; d < hd; d += 4) {
          const float4 k4 = four(keys + key * row + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 q4 = four(q_s + (r0 + i) * ld + d);
            s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
          }
        }
        bool sees[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sees[i] = token[i] >= 0 && at + key <= high[i] && at + key >= low[i] && has_page(p, who, token[i]);
          s[i] = sees[i] ? s[i] * scale : -INFINITY;
          const float top = warp_max(s[i]);
          if (lane == 0) sm_max[it & 1][warp >> 2][r0 + i] = top;
        }
        __syncthreads();
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float top = fmaxf(m[i], fmaxf(sm_max[it & 1][0][r0 + i], sm_max[it & 1][1][r0 + i]));
          const float shift = top > -INFINITY ? top : 0.f;
          const float fade = m[i] > -INFINITY ? exp2f(m[i] - shift) : 1.f;
          m[i] = top;
          // (a masked key's weight is marked by -1: its value is not multiplied)
          w[i] = sees[i] ? exp2f(s[i] - shift) : -1.f;
          l[i] = l[i] * fade + (sees[i] ? w[i] : 0.f);
          if (key == 0) sm_fade[r0 + i] = fade;
        }
        *reinterpret_cast<float4*>(sm_p + key * FMA_LD + r0) = make_float4(w[0], w[1], w[2], w[3]);
        __syncthreads();
        if (group < n_groups) {
          const float4 f = four(sm_fade + s0);
          const float fades[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[i].x *= fades[i]; acc[i].y *= fades[i]; acc[i].z *= fades[i]; acc[i].w *= fades[i];
          }
          for (int k = group; k < PAGE; k += n_groups) {
            const float4 v = four(vals + k * row + d4), weights = four(sm_p + k * FMA_LD + s0);
            const float each_w[4] = {weights.x, weights.y, weights.z, weights.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (each_w[i] != -1.f) {
                acc[i].x = fmaf(each_w[i], v.x, acc[i].x);
                acc[i].y = fmaf(each_w[i], v.y, acc[i].y);
                acc[i].z = fmaf(each_w[i], v.z, acc[i].z);
                acc[i].w = fmaf(each_w[i], v.w, acc[i].w);
              }
          }
        }
        __syncthreads();
        if (stages == 1) {
          if (it + 1 < count) bring(it + 1);
          cp_async_commit();
        }
      }
      cp_async_wait<0>();
      __syncthreads();
    }
    // the groups of keys together, in order; sums over a row's keys
    if (group < n_groups)
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(groups_s + (size_t)(group * FMA_ROWS + s0 + i) * ld + d4) = acc[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sum = warp_sum(l[i]);
      if (lane == 0) sm_l[warp >> 2][r0 + i] = sum;
    }
    __syncthreads();
    for (int i = tid; i < FMA_ROWS * fours; i += FMA_THREADS) {
      const int r = i / fours, d = (i % fours) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int g = 0; g < n_groups; ++g) {
        const float4 y = four(groups_s + (size_t)(g * FMA_ROWS + r) * ld + d);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      *reinterpret_cast<float4*>(q_s + r * ld + d) = x;
    }
    if (lane == 0 && warp < 4)
#pragma unroll
      for (int i = 0; i < 4; ++i) sm_ml[r0 + i] = make_float2(m[i], sm_l[0][r0 + i] + sm_l[1][r0 + i]);
  } else {
    if (tid < FMA_ROWS) sm_ml[tid] = make_float2(-INFINITY, 0.f);
  }
  finish<T, FMA_ROWS>(p, a, q_s, ld, sm_ml);
}

// ---- launch shapes -------------------------------------------------------------------------------------------------
enum { FMA, MMA, TCGEN05 };
struct Shape { int kind, rows, tiles, splits, cluster; bool several; };  // several: two blocks of a multiprocessor

Shape shape_of(int dtype, int heads, int kv_heads, int head_dim, int groups, int max_rows, int max_context) {
  Shape s;
  const int query_rows = max_rows * (heads / kv_heads), pages = (max_context + PAGE - 1) / PAGE;
  const bool tensor = dtype == DLLM_BF16 && head_dim % 16 == 0 && head_dim <= 128;
  // (tcgen05 against mma.sync with heads of 64 and 128, us: 1 x 4 beams on 110 positions, 9 heads on 3, 9.3 and 8.9; eight new tokens, 32
  // heads on 8, on 2,000 positions 10.5 and 14.4, 10.7 and 19.5, on 80,000 41 and 84, 61 and 129)
  s.kind = !tensor ? FMA : head_dim >= 64 ? TCGEN05 : MMA;
  if (s.kind == FMA) s.rows = FMA_ROWS;
  else if (s.kind == MMA) s.rows = query_rows <= 16 ? 16 : query_rows <= 32 ? 32 : 64;
  else s.rows = query_rows <= 32 ? 32 : 64;
  s.tiles = (query_rows + s.rows - 1) / s.rows;
  // Blocks of a tile and kv head: as many as fill the device, but not more than there can be pages, in the largest clusters that
  // do not cost more than a fifth of them; where there are at most 64 pages one cluster, which needs no scratch and no second
  // round (by multiply-adds, where a page costs more, at most 16: 9 heads on 3 of 64, 2 x 5 beams on 700 positions, one cluster
  // of 8 18.0 us, three of 7 14.9; 4 x 4 on 2,000 28.5 and 20.8).
  // Eight new tokens a prompt, 32 heads on 8 of 128, us with one cluster of 8, 4 of 4, 9 of 2 and 18 of 1: 2,000 positions 13.4, 17.2,
  // 20.7, 24.1; 80,000: -, 62.6, 65.9, 70.1. Sizes that are no powers of two: three prompts of 20,000 positions 46.8 with three
  // clusters of 2, 44.0 with one of 5; five of 10,000 43.8 with three of 1, 38.7 with one of 3; 2 x 8 beams on 2,000 16.1 with
  // one of 4, 13.6 with one of 6.
  // RESIDENT: clusters of 1 to 8 blocks that start together, one and two blocks a multiprocessor. A cluster lies within a part of
  // the device, and what is left over of a part stays idle; the last few that would fit start late behind another kernel's blocks
  // (float32, two blocks, clusters of 8: 31 of them 28.4 us, 33 36.2).
  static const int RESIDENT[2][MAX_CLUSTER] = {{148, 74, 44, 33, 25, 22, 15, 15}, {296, 148, 90, 70, 54, 44, 36, 31}};
  const long long pairs = (long long)groups * s.tiles * kv_heads, most = pages + (s.kind == FMA ? 2 : 1) * max_rows;
  // (Two blocks for heads of 64 and 32 rows where there are more pairs than multiprocessors: 32 heads on 32, 8 x 4 beams on 60, 1,000,
  // 2,000 and 4,000 positions 20.0, 30.7, 37.7, 53.5 us with one, 13.6, 25.1, 36.4, 56.0 with two; 16 x 4 on 1,000 and 4,000 57.6, 104 and
  // 43.8, 91.7.)
  s.several = s.kind == MMA || (s.kind == FMA && head_dim * (dtype == DLLM_BF16 ? 2 : 4) <= 256) ||
              (s.kind == TCGEN05 && head_dim == 64 && s.rows == 32 && pairs > 148);
  long long blocks[MAX_CLUSTER], best = 0;
  for (int c = 1; c <= MAX_CLUSTER; ++c) {
    long long n = RESIDENT[s.several][c - 1] / pairs;
    if (n > MAX_CLUSTERS) n = MAX_CLUSTERS;
    if ((s.kind == FMA ? most <= 16 : pages <= 64) && n > 1) n = c > 1 ? 1 : 0;
    if (n * c > most) n = most / c;
    blocks[c - 1] = n * c;
    if (n * c > best) best = n * c;
  }
  s.splits = s.cluster = 1;
  for (int c = 1; c <= MAX_CLUSTER; ++c)
    if (blocks[c - 1] > 0 && blocks[c - 1] * 5 >= best * 4) { s.cluster = c; s.splits = (int)blocks[c - 1]; }
  return s;
}

template <int HD, int MT, int WM, int STAGES>
int launch_mma(const Args& a, dim3 grid, cudaStream_t stream) {
  constexpr int ROWS = 16 * MT * WM;
  constexpr int ring = STAGES * 2 * 64 * HD * 2, sums = 4 * ROWS * HD * 4;
  constexpr int smem = ROWS * HD * 2 + (ring > sums ? ring : sums);
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)mma_kernel<HD, MT, WM, STAGES>, smem, done)) return DLLM_LAUNCH_FAILED;
  return launch_clusters(mma_kernel<HD, MT, WM, STAGES>, grid, WM * 128, smem, a.cluster, stream, a);
}

template <typename T>
int launch_fma(const Args& a, dim3 grid, cudaStream_t stream) {
  const int hd = a.cache.head_dim, rows = FMA_ROWS * (hd + 4) * 4;
  const int ring = fma_stages<T>(hd) * 2 * PAGE * fma_row<T>(hd) * (int)sizeof(T);
  const int each = hd, n = FMA_THREADS / each < 16 ? FMA_THREADS / each : 16;  // (groups of keys, of hd / 4 x 4 threads)
  const int sums = n * FMA_ROWS * (hd + 4) * 4;
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)fma_kernel<T>, FMA_MOST, done)) return DLLM_LAUNCH_FAILED;
  return launch_clusters(fma_kernel<T>, grid, FMA_THREADS, rows + (ring > sums ? ring : sums), a.cluster, stream, a);
}
}  // namespace

// Query rows of a tile in the low 16 bits, clusters above: scratch holds groups x tiles x kv_heads x clusters x rows x
// (head_dim + 2) floats where there is more than one, tickets groups x tiles x kv_heads x 8 words.
DLLM_EXPORT int dllm_attention_shared_shape(int dtype, int heads, int kv_heads, int head_dim, int groups, int max_rows,
                                            int max_context) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || groups <= 0 || max_rows <= 0 || max_context <= 0) return DLLM_BAD_ARGUMENT;
  Shape s = shape_of(dtype, heads, kv_heads, head_dim, groups, max_rows, max_context);
  return s.rows | s.splits / s.cluster << 16;
}

// See the head of the file. out, q [tokens, heads * head_dim] in the cache's type; slots, positions: each token's table row and
// position; cuts [groups + 1]: the groups' first tokens; shared [groups]: pages from the first on that a group's table rows have
// in common; the cache entry has `pages` pages. One structure, `bytes` long, which the caller packs at once.
struct DllmAttentionShared {
  void* out;
  const void* q;
  void* base;
  const int *page_table, *slots, *positions, *cuts, *shared;
  float* scratch;
  unsigned* tickets;
  int* status;
  cudaStream_t stream;
  long long pages;
  int tokens, max_pages, page_size, dtype, heads, kv_heads, head_dim, groups, max_rows, max_context, window;
  float scale;
};
DLLM_EXPORT int dllm_attention_shared(const DllmAttentionShared* call, int bytes) {
  if (bytes != (int)(offsetof(DllmAttentionShared, scale) + sizeof(float))) return DLLM_BAD_ARGUMENT;
  const DllmAttentionShared& c = *call;
  const int dtype = c.dtype, heads = c.heads, kv_heads = c.kv_heads, head_dim = c.head_dim, groups = c.groups, max_rows = c.max_rows,
            max_context = c.max_context;
  if (groups <= 0 || max_rows <= 0) return DLLM_OK;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_context <= 0 || c.window < 0 || c.pages <= 0) return DLLM_BAD_ARGUMENT;
  if (head_dim % 8 || head_dim <= 0 || head_dim > FMA_DIM || c.page_size != PAGE || kv_heads > 65535 ||
      ((uintptr_t)c.out | (uintptr_t)c.q | (uintptr_t)c.base) & 15)
    return DLLM_UNSUPPORTED_SIZE;
  Shape s = shape_of(dtype, heads, kv_heads, head_dim, groups, max_rows, max_context);
  if ((long long)groups * s.tiles > 65535) return DLLM_UNSUPPORTED_SIZE;
  if (s.splits > s.cluster && (!c.scratch || !c.tickets)) return DLLM_BAD_ARGUMENT;
  if (s.splits > s.cluster && ((uintptr_t)c.scratch & 15)) return DLLM_UNSUPPORTED_SIZE;  // (fours of floats go there)
  Args a{c.out, c.q, KvLayout{c.base, c.page_table, c.max_pages, c.page_size, kv_heads, head_dim}, c.slots, c.positions, c.cuts,
         c.shared, c.scratch, c.tickets, c.status, heads, c.window, s.tiles, s.splits, s.cluster, c.tokens, max_rows, c.scale};
  const long long pages = c.pages;
  cudaStream_t stream = c.stream;
  dim3 grid(s.splits, kv_heads, groups * s.tiles);
  if (s.kind == FMA) return dtype == DLLM_BF16 ? launch_fma<bf16>(a, grid, stream) : launch_fma<float>(a, grid, stream);
  if (s.kind == TCGEN05) {
    if (pages * 2 * kv_heads * PAGE > 0x7fffffffll) return DLLM_UNSUPPORTED_SIZE;  // (a TMA coordinate is an int)
    if (head_dim > 64) return s.rows == 32 ? t5::launch<2, 32, 2>(a, pages, grid, stream) : t5::launch<2, 64, 1>(a, pages, grid, stream);
    if (s.rows == 64) return t5::launch<1, 64, 1>(a, pages, grid, stream);
    return s.several ? t5::launch<1, 32, 1>(a, pages, grid, stream) : t5::launch<1, 32, 3>(a, pages, grid, stream);
  }
  if (head_dim <= 32) {
    if (s.rows == 16) return launch_mma<32, 1, 1, 4>(a, grid, stream);
    if (s.rows == 32) return launch_mma<32, 2, 1, 4>(a, grid, stream);
    return launch_mma<32, 2, 2, 4>(a, grid, stream);
  }
  if (s.rows == 16) return launch_mma<64, 1, 1, 4>(a, grid, stream);  // (heads of 48)
  if (s.rows == 32) return launch_mma<64, 2, 1, 4>(a, grid, stream);
  return launch_mma<64, 2, 2, 4>(a, grid, stream);
}
