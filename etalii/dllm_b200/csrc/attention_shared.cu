// Attention of a few new tokens a group over the paged cache, where the tokens of a group share pages: the beams of one
// prompt (the prompt's pages in common, pages of their own behind them), or the tokens of a short chunk that is appended to
// one sequence (all pages in common, each token sees up to itself). Pages in common are read once for all tokens of the
// group and all query heads of the key/value head; the others once for each token.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max),  over the positions j <= position of the token's own
//   table row (and j > position - window). A token at position -1 sees nothing: zeros.
//
// A group's query rows (tokens x query heads of one kv head, in that order) are cut into tiles of ROWS. What a tile has to read is
// a list of pages: those in common, then each token's own. The list is cut into `splits` stretches of equal length, a block
// each, so that the device is filled whatever the contexts are; running maximum and sum are kept in float32. Partial results go to
// scratch, and the block that finishes last for its tile and kv head (a ticket; nobody waits) joins them in order.
//
// bfloat16, head sizes that are multiples of 16 up to 128: tensor cores (mma.sync). Pages travel by cp.async through a
// ring of stages; the four warps that share a tile's rows take 16 of a page's 64 keys each, with a maximum and a sum of
// their own, so that no page costs a barrier between softmax and product. Probabilities are rounded to bfloat16 as the second
// product's operand. Everything else (float32, other head sizes): fused multiply-adds on pages in shared memory.
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
constexpr int MAX_SPLITS = 128;
constexpr int FULL = 0x7fffffff;
constexpr int TOO_MANY = 51;    // status: a group has more tokens than the launch was told

struct Args {
  void* out;
  const void* q;
  KvLayout cache;
  const int *slots, *positions, *cuts, *shared;
  float* scratch;      // [tile, kv head][split][ROWS][head_dim], then [..][ROWS][2]
  unsigned* tickets;   // one a (tile, kv head), zero between launches
  int* status;
  int heads, window, tiles, splits;
  float scale;
};

// What a tile's block works on: the same in every block of the tile.
struct Plan {
  int token0, tokens;            // the tile's tokens
  int row0, rows;                // its query rows, counted from the group's first
  int shared_first, shared_count, total;
  int longest;                   // the token that sees furthest: its table row names the pages in common
  int all_from, all_to;          // positions that every token sees
  int position[MAX_ROWS], low[MAX_ROWS], slot[MAX_ROWS];   // of each token: it sees low .. position
  int own_first[MAX_ROWS], own_base[MAX_ROWS + 1];         // its pages behind those in common: first, place in the list
  int page[LIST], at[LIST], whose[LIST];                   // a stretch of the list: page, first position, token or -1
  int last;
};

// Fills the plan (all threads call; ends with a barrier).
__device__ __forceinline__ void make_plan(Plan& p, const Args& a, int rows_per_tile) {
  const int group = blockIdx.z / a.tiles, tile = blockIdx.z % a.tiles;
  const int per_kv = a.heads / a.cache.kv_heads;
  const int first = a.cuts[group], count = a.cuts[group + 1] - first;
  const int row0 = tile * rows_per_tile, rows = min(rows_per_tile, count * per_kv - row0);
  if (threadIdx.x == 0 && tile == a.tiles - 1 && count * per_kv > a.tiles * rows_per_tile)
    *reinterpret_cast<volatile int*>(a.status) = TOO_MANY;  // (the launch was made for fewer tokens a group)
  if (rows <= 0) {
    if (threadIdx.x == 0) { p.rows = 0; p.total = 0; }
    __syncthreads();
    return;
  }
  const int t0 = row0 / per_kv, tokens = (row0 + rows - 1) / per_kv - t0 + 1;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int shared = a.shared[group];
    int furthest = -1, which = 0, least_first = FULL, from = 0, to = FULL;
    constexpr int EACH = MAX_ROWS / 32;
    int pos[EACH], low[EACH], pages[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      int t = lane + 32 * u;
      pos[u] = -1;
      low[u] = 0;
      int slot = 0;
      if (t < tokens) {
        pos[u] = a.positions[first + t0 + t];
        slot = a.slots[first + t0 + t];
        if (slot < 0) { slot = 0; pos[u] = -1; }
        pos[u] = min(pos[u], a.cache.max_pages * PAGE - 1);
        low[u] = a.window > 0 ? max(0, pos[u] + 1 - a.window) : 0;
        from = max(from, low[u]);
        to = min(to, pos[u]);
        p.position[t] = pos[u];
        p.low[t] = low[u];
        p.slot[t] = slot;
      }
      pages[u] = pos[u] / PAGE + 1;
      if (pos[u] < 0) pages[u] = 0;
      if (pos[u] > furthest) { furthest = pos[u]; which = t; }
      if (pages[u]) least_first = min(least_first, low[u] / PAGE);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      int f = __shfl_xor_sync(0xffffffffu, furthest, o), w = __shfl_xor_sync(0xffffffffu, which, o);
      if (f > furthest || (f == furthest && w < which)) { furthest = f; which = w; }
      least_first = min(least_first, __shfl_xor_sync(0xffffffffu, least_first, o));
      from = max(from, __shfl_xor_sync(0xffffffffu, from, o));
      to = min(to, __shfl_xor_sync(0xffffffffu, to, o));
    }
    const int common = min(max(shared, 0), furthest < 0 ? 0 : furthest / PAGE + 1);
    const int shared_count = max(0, common - least_first);
    int own[EACH], first_own[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      first_own[u] = max(common, low[u] / PAGE);
      own[u] = max(0, pages[u] - first_own[u]);
    }
    int base[EACH], sum = 0;  // places in the list, tokens in order: lanes hold t, t + 32, ..
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      int through = own[u];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        int other = __shfl_up_sync(0xffffffffu, through, o);
        if (lane >= o) through += other;
      }
      base[u] = sum + through - own[u];
      sum += __shfl_sync(0xffffffffu, through, 31);
      int t = lane + 32 * u;
      if (t < tokens) { p.own_first[t] = first_own[u]; p.own_base[t] = shared_count + base[u]; }
    }
    if (lane == 0) {
      p.token0 = first + t0;
      p.tokens = tokens;
      p.row0 = row0;
      p.rows = rows;
      p.shared_first = least_first;
      p.shared_count = shared_count;
      p.total = shared_count + sum;
      p.own_base[tokens] = shared_count + sum;
      p.longest = which;
      p.all_from = from;
      p.all_to = to;
    }
  }
  __syncthreads();
}

// Place i of the plan's list: whose page it is (-1: the group's) and its index in the table row.
__device__ __forceinline__ int look_up(const Plan& p, int i, int& whose) {
  whose = -1;
  if (i < p.shared_count) return p.shared_first + i;
  int lo = 0, hi = p.tokens - 1;  // the last token whose own pages begin at or before i
  while (lo < hi) {
    int mid = (lo + hi + 1) >> 1;
    if (p.own_base[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  whose = lo;
  return p.own_first[lo] + i - p.own_base[lo];
}
__device__ __forceinline__ int page_of(const Plan& p, const Args& a, int whose, int index) {
  return a.cache.page_table[(size_t)p.slot[whose < 0 ? p.longest : whose] * a.cache.max_pages + index];
}

// Lists the pages [begin, end) of the plan's list (at most LIST of them). All threads call; ends with a barrier.
__device__ __forceinline__ void list_pages(Plan& p, const Args& a, int begin, int end) {
  for (int i = begin + (int)threadIdx.x; i < end; i += blockDim.x) {
    int whose, index = look_up(p, i, whose);
    p.page[i - begin] = page_of(p, a, whose, index);
    p.at[i - begin] = index * PAGE;
    p.whose[i - begin] = whose;
  }
  __syncthreads();
}

// The last block of a tile and kv head joins the partial results of all splits, in order. weight: ROWS x splits floats of shared memory.
template <typename T, int ROWS, int THREADS>
__device__ __forceinline__ void join(const Plan& p, const Args& a, size_t pair, float* weight) {
  const int hd = a.cache.head_dim, splits = a.splits, per_kv = a.heads / a.cache.kv_heads;
  const float* part = a.scratch + pair * splits * ROWS * hd;
  const float* ml = a.scratch + (size_t)gridDim.z * gridDim.y * splits * ROWS * hd + pair * splits * ROWS * 2;
  auto empty = [&](int s) { return (long long)p.total * s / splits == (long long)p.total * (s + 1) / splits; };
  for (int r = threadIdx.x; r < p.rows; r += THREADS) {
    float top = -INFINITY, sum = 0.f;
    for (int s = 0; s < splits; ++s)
      if (!empty(s)) top = fmaxf(top, __ldcg(ml + (s * ROWS + r) * 2));
    for (int s = 0; s < splits; ++s) {
      float w = 0.f;
      if (!empty(s)) {
        float2 pair_ml = __ldcg(reinterpret_cast<const float2*>(ml + (s * ROWS + r) * 2));
        w = pair_ml.x > -INFINITY ? exp2f(pair_ml.x - top) : 0.f;
        if (pair_ml.x > -INFINITY || pair_ml.y != 0.f) sum += pair_ml.x > -INFINITY ? w * pair_ml.y : pair_ml.y;
      }
      weight[s * ROWS + r] = w;
    }
    weight[splits * ROWS + r] = sum != 0.f ? 1.f / sum : 0.f;
  }
  __syncthreads();
  const int pieces = hd / 4;
  for (int i = threadIdx.x; i < p.rows * pieces; i += THREADS) {
    int r = i / pieces, d = (i % pieces) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
      float w = weight[s * ROWS + r];
      if (w == 0.f) continue;
      float4 v = __ldcg(reinterpret_cast<const float4*>(part + ((size_t)s * ROWS + r) * hd + d));
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    }
    float inv = weight[splits * ROWS + r];
    int row = p.row0 + r, token = p.token0 + row / per_kv - p.row0 / per_kv, head = blockIdx.y * per_kv + row % per_kv;
    T* to = static_cast<T*>(a.out) + ((size_t)token * a.heads + head) * hd + d;
    to[0] = from_float<T>(acc.x * inv);
    to[1] = from_float<T>(acc.y * inv);
    to[2] = from_float<T>(acc.z * inv);
    to[3] = from_float<T>(acc.w * inv);
  }
}

// Is this block the last of its tile and kv head? (All threads call.)
__device__ __forceinline__ bool is_last(Plan& p, const Args& a, size_t pair) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    p.last = atomicAdd(&a.tickets[pair], 1u) == (unsigned)(a.splits - 1);
    if (p.last) a.tickets[pair] = 0u;
  }
  __syncthreads();
  __threadfence();
  return p.last != 0;
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
// one of two packed bfloat16 is not finite
__device__ __forceinline__ bool odd_pair(unsigned v) {
  return (v & 0x7f80u) == 0x7f80u || (v & 0x7f800000u) == 0x7f800000u;
}
// where piece `c` (16 bytes) of row r lies: neighbouring rows' pieces in different banks
template <int HD> __device__ __forceinline__ int place(int r, int c) {
  return r * HD + 8 * (HD >= 64 ? c ^ (r & 7) : c ^ ((r >> 1) & 3));
}

// HD: the head size, padded (32, 64, 128). A warp has 16 * MT query rows; WM warps (of 4) lie one above another in the tile.
template <int HD, int MT, int WM, int STAGES>
__global__ void __launch_bounds__(WM * 128) mma_kernel(const Args a) {
  constexpr int THREADS = WM * 128, ROWS = 16 * MT * WM;
  constexpr bool KEEP_Q = MT * HD <= 128;  // the queries' operands stay in registers
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ Plan p;
  __shared__ float sm_m[4][ROWS], sm_l[4][ROWS];
  bf16* q_s = reinterpret_cast<bf16*>(smem_raw);  // [ROWS][HD]
  bf16* ring = q_s + ROWS * HD;                    // per stage: keys [64][HD], values [64][HD]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int quarter = warp & 3, tier = warp >> 2;  // which 16 keys of a page; which of the tile's rows
  const int hd = a.cache.head_dim, pieces = hd >> 3, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  make_plan(p, a, ROWS);
  if (p.rows == 0) return;
  const size_t pair = (size_t)blockIdx.z * gridDim.y + kv;
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  if (begin < end || a.splits == 1) {
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
        high[i][e] = real ? p.position[t] : FULL;
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
      list_pages(p, a, part, part + count);
      auto bring = [&](int i) {
        bf16* keys = ring + (size_t)(i % STAGES) * 2 * 64 * HD;
        int page = p.page[i], at = p.at[i], whose = p.whose[i];
        // what nobody sees is not read: zeros lie there
        int from = whose < 0 ? at : p.low[whose], to = whose < 0 ? p.position[p.longest] : p.position[whose];
        const bf16* src = base + kv_offset(a.cache, page, 0, kv, 0);
        const size_t values = (size_t)a.cache.kv_heads * PAGE * hd;
        for (int c = tid; c < 64 * (HD / 8); c += THREADS) {
          int r = c / (HD / 8), d = c % (HD / 8);
          bool ok = at + r >= from && at + r <= to;
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
        const int whose = p.whose[it], at = p.at[it] + 16 * quarter;
        const bool whole = whose < 0 && at >= p.all_from && at + 15 <= p.all_to;
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
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                float v = s[i][j][2 * e + u] * scale;
                if (!whole) {
                  int key = at + 8 * j + 2 * (lane & 3) + u;
                  bool sees = key <= high[i][e] && key >= low[i][e] && (whose < 0 || whose == token[i][e]);
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
#pragma unroll
          for (int n = 0; n < HD / 16; ++n) {
            unsigned vf[4];
            ldmatrix_x4_trans(vf, vals + place<HD>(16 * quarter + (lane & 15), 2 * n + (lane >> 4)));
            odd = odd || odd_pair(vf[0]) || odd_pair(vf[1]) || odd_pair(vf[2]) || odd_pair(vf[3]);
          }
          odd = __any_sync(0xffffffffu, odd);
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
        l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 1);
        l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 2);
        int r = 16 * (MT * tier + i) + (lane >> 2) + 8 * e;
        if ((lane & 3) == 0) { sm_m[quarter][r] = m[i][e]; sm_l[quarter][r] = l[i][e]; }
      }
    __syncthreads();
    float* sum = reinterpret_cast<float*>(ring);  // [4][ROWS][HD]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int r = 16 * (MT * tier + i) + (lane >> 2) + 8 * e;
        float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
        float w = m[i][e] > -INFINITY ? exp2f(m[i][e] - top) : 0.f;
        // (rows without a key in this quarter: nothing, whatever the products made of zeros)
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          float2 v = make_float2(0.f, 0.f);
          if (w != 0.f) v = make_float2(o[i][n][2 * e] * w, o[i][n][2 * e + 1] * w);
          *reinterpret_cast<float2*>(sum + ((size_t)quarter * ROWS + r) * HD + 8 * n + 2 * (lane & 3)) = v;
        }
      }
    __syncthreads();
    const int fours = hd / 4;
    for (int i = tid; i < p.rows * fours; i += THREADS) {
      int r = i / fours, d = (i % fours) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, sm_m[w][r]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float4 x = *reinterpret_cast<const float4*>(sum + ((size_t)w * ROWS + r) * HD + d);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        total += sm_m[w][r] > -INFINITY ? sm_l[w][r] * exp2f(sm_m[w][r] - top) : sm_l[w][r];
      }
      if (a.splits == 1) {
        float inv = total != 0.f ? 1.f / total : 0.f;
        int row = p.row0 + r, t = p.token0 + row / per_kv - p.row0 / per_kv;
        uint2 packed = make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
        *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + ((size_t)t * a.heads + kv * per_kv + row % per_kv) * hd + d) = packed;
      } else {
        float* part = a.scratch + ((pair * a.splits + blockIdx.x) * ROWS + r) * hd + d;
        *reinterpret_cast<float4*>(part) = v;
        if (d == 0) {
          float* ml = a.scratch + (size_t)gridDim.z * gridDim.y * a.splits * ROWS * hd + ((pair * a.splits + blockIdx.x) * ROWS + r) * 2;
          *reinterpret_cast<float2*>(ml) = make_float2(top, total);
        }
      }
    }
  }
  if (a.splits == 1) return;
  if (is_last(p, a, pair)) join<bf16, ROWS, THREADS>(p, a, pair, reinterpret_cast<float*>(smem_raw));
}

// ---- 5th-generation tensor cores -----------------------------------------------------------------------------------
// Scores and outputs in tensor memory, pages by TMA. A product has 128 rows whatever the tile has, so a tile of at most
// 32 (64) query rows stands in it COPIES = 4 (2) times, one copy above the other, and every copy works on its own 16 (32) of
// a page's 64 keys: the P tile has the probabilities of those and zeros elsewhere, and the copies' outputs are added at the end.
// All four warps of a softmax group are then busy with a page, and a thread has 64 / COPIES scores of one query row.
//   warps 0..7  two softmax groups that take the pages in turn, each with scores, P and outputs of its own: scores from tensor
//               memory, mask, running maximum (renewed only when a score exceeds it by 2^8) and sum, P as bfloat16 into the
//               swizzled tile, outputs scaled in tensor memory when the maximum is renewed.
//   warp 8      looks pages up, 32 at a time, and issues their TMA loads; warp 9 issues the scores' products, warp 10 the outputs'.
// Pages that some row sees in part are looked at: one with a value that is not finite is added by the softmax warps, key by key,
// and its product left out.
// Every wait is bounded; a role that gives up sets the status word and leaves.
namespace t5 {
using namespace tc5;
constexpr int GROUPS = 2, SOFT_WARPS = 4 * GROUPS, THREADS = (SOFT_WARPS + 3) * 32;
constexpr int P_BYTES = 128 * 128;

template <int BOXES> struct Shape {
  static constexpr int K_STAGES = BOXES == 2 ? 4 : 3, V_STAGES = BOXES == 2 ? 5 : 4;
  static constexpr int Q_BYTES = BOXES * 128 * 128, KV_BYTES = BOXES * 64 * 128;
  static constexpr int OUT = BOXES * 64;                       // columns of the outputs
  static constexpr unsigned COLUMNS = BOXES == 2 ? 512 : 256;  // of tensor memory
  static constexpr int SMEM = Q_BYTES + GROUPS * P_BYTES + (K_STAGES + V_STAGES) * KV_BYTES + 1024;
  static constexpr int LD = OUT + 4;  // floats of a row of the exchange at the end, which lies in P's and the stages' place
  static_assert(GROUPS * (64 + OUT) <= (int)COLUMNS, "tensor memory");
  static_assert(GROUPS * 128 * LD * 4 <= GROUPS * P_BYTES + (K_STAGES + V_STAGES) * KV_BYTES, "exchange");
};

struct Barriers {
  uint64_t k_full[5], k_empty[5], v_full[5], v_empty[5], s_full[GROUPS], s_empty[GROUPS], p_full[GROUPS], o_full[GROUPS];
};

template <int BOXES, int COPIES>
__global__ void __launch_bounds__(THREADS, BOXES == 1 ? 2 : 1) kernel(const __grid_constant__ CUtensorMap map_kv, const Args a) {
  typedef Shape<BOXES> S;
  constexpr int ROWS = 128 / COPIES, KEYS = 64 / COPIES;
  constexpr int K_STAGES = S::K_STAGES, V_STAGES = S::V_STAGES, KV_BYTES = S::KV_BYTES;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned char* tiles = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);  // swizzle atoms: 1 KB
  unsigned char* q_s = tiles;
  unsigned char* p_s = q_s + S::Q_BYTES;
  unsigned char* k_s = p_s + GROUPS * P_BYTES;
  unsigned char* v_s = k_s + K_STAGES * KV_BYTES;
  __shared__ Plan p;
  __shared__ Barriers bar;
  __shared__ unsigned tmem_base_s;
  __shared__ float sm_m[GROUPS][128], sm_l[GROUPS][128];
  __shared__ int odd_s[GROUPS], skip_s[GROUPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = a.cache.head_dim, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads;
  pdl_launch_dependents();
  if (tid == 0) {
    for (int s = 0; s < K_STAGES; ++s) { mbar_init(&bar.k_full[s], 1); mbar_init(&bar.k_empty[s], 1); }
    for (int s = 0; s < V_STAGES; ++s) { mbar_init(&bar.v_full[s], 1); mbar_init(&bar.v_empty[s], 1); }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.s_empty[i], 4);
      mbar_init(&bar.p_full[i], 4);
      mbar_init(&bar.o_full[i], 1);
      odd_s[i] = skip_s[i] = 0;
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_kv) : "memory");
  }
  if (COPIES > 1)  // (what P never gets a value for is zero)
    for (int i = tid; i < GROUPS * P_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(p_s)[i] = make_uint4(0u, 0u, 0u, 0u);
  pdl_wait();
  make_plan(p, a, ROWS);
  if (p.rows == 0) return;
  const size_t pair = (size_t)blockIdx.z * gridDim.y + kv;
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  const int steps = end - begin;
  if (steps > 0 || a.splits == 1) {
    if (warp == SOFT_WARPS + 1) tmem_alloc(&tmem_base_s, S::COLUMNS);
    {  // the queries, once a copy; rows beyond the tile and dimensions beyond the head are zeros
      const bf16* q = static_cast<const bf16*>(a.q);
      for (int i = tid; i < ROWS * BOXES * 8; i += THREADS) {
        int r = i / (BOXES * 8), c = i % (BOXES * 8), row = p.row0 + r;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < p.rows && c * 8 < hd)
          v = *reinterpret_cast<const uint4*>(q + ((size_t)(p.token0 + row / per_kv - p.row0 / per_kv) * a.heads + kv * per_kv + row % per_kv) * hd + c * 8);
#pragma unroll
        for (int copy = 0; copy < COPIES; ++copy) {
          int at = copy * ROWS + r;
          *reinterpret_cast<uint4*>(q_s + (c >> 3) * 16384 + at * 128 + (((c & 7) ^ (at & 7)) << 4)) = v;
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const unsigned tmem_s = tmem_base_s, tmem_o = tmem_base_s + GROUPS * 64;
    if (warp == SOFT_WARPS) {
      int issued_k = 0, issued_v = 0;
      bool ok = true;
      for (int j0 = 0; j0 < steps && ok; j0 += 32) {
        int page = 0;
        if (j0 + lane < steps) {
          int whose, index = look_up(p, begin + j0 + lane, whose);
          page = page_of(p, a, whose, index);
        }
        for (int u = 0; u < 32 && j0 + u < steps && ok; ++u) {
          const int j = j0 + u, sk = j % K_STAGES, sv = j % V_STAGES;
          const int at = __shfl_sync(0xffffffffu, page, u);
          if (lane == 0) {
            const int row_k = ((at * 2 + 0) * a.cache.kv_heads + kv) * PAGE, row_v = ((at * 2 + 1) * a.cache.kv_heads + kv) * PAGE;
            if (j >= K_STAGES && !mbar_wait(&bar.k_empty[sk], (j / K_STAGES - 1) & 1)) ok = false;
            if (ok) {
              mbar_expect_tx(&bar.k_full[sk], KV_BYTES);
#pragma unroll
              for (int x = 0; x < BOXES; ++x) tma_load_2d(k_s + sk * KV_BYTES + x * 8192, &map_kv, &bar.k_full[sk], x * 64, row_k);
              issued_k = j + 1;
              if (j >= V_STAGES && !mbar_wait(&bar.v_empty[sv], (j / V_STAGES - 1) & 1)) ok = false;
            }
            if (ok) {
              mbar_expect_tx(&bar.v_full[sv], KV_BYTES);
#pragma unroll
              for (int x = 0; x < BOXES; ++x) tma_load_2d(v_s + sv * KV_BYTES + x * 8192, &map_kv, &bar.v_full[sv], x * 64, row_v);
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
        constexpr unsigned idesc = instr_desc(128, 64);
        const unsigned q_addr = smem_u32(q_s);
        for (int i = 0; i < steps; ++i) {
          const int g = i % GROUPS, s = i % K_STAGES;
          if (!mbar_wait(&bar.k_full[s], (i / K_STAGES) & 1) || (i >= GROUPS && !mbar_wait(&bar.s_empty[g], (i / GROUPS - 1) & 1))) {
            *(volatile int*)a.status = 53;
            break;
          }
          fence_after_sync();
          const unsigned k_addr = smem_u32(k_s + s * KV_BYTES);
#pragma unroll
          for (int k = 0; k < BOXES * 4; ++k)
            if (k * 16 < hd)
              umma(tmem_s + (unsigned)(g * 64), smem_desc(q_addr + (k >> 2) * 16384 + (k & 3) * 32),
                   smem_desc(k_addr + (k >> 2) * 8192 + (k & 3) * 32), idesc, k > 0 ? 1u : 0u);
          tcgen05_commit(&bar.k_empty[s]);
          tcgen05_commit(&bar.s_full[g]);
        }
      }
    } else if (warp == SOFT_WARPS + 2) {
      if (lane == 0) {
        constexpr unsigned idesc = instr_desc(128, 64, true);
        for (int i = 0; i < steps; ++i) {
          const int g = i % GROUPS, s = i % V_STAGES;
          if (!mbar_wait(&bar.p_full[g], (i / GROUPS) & 1) || !mbar_wait(&bar.v_full[s], (i / V_STAGES) & 1)) {
            *(volatile int*)a.status = 54;
            break;
          }
          fence_after_sync();
          if (!*(volatile int*)&skip_s[g]) {
            const unsigned p_addr = smem_u32(p_s + g * P_BYTES), v_addr = smem_u32(v_s + s * KV_BYTES);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int x = 0; x < BOXES; ++x)
                umma(tmem_o + (unsigned)(g * S::OUT + x * 64), smem_desc(p_addr + k * 32), smem_desc(v_addr + x * 8192 + k * 2048), idesc,
                     (k > 0 || i >= GROUPS) ? 1u : 0u);
          }
          tcgen05_commit(&bar.v_empty[s]);
          tcgen05_commit(&bar.o_full[g]);
        }
      }
    } else {
      const int g = warp >> 2, r = (warp & 3) * 32 + lane, row = r % ROWS, first_key = r / ROWS * KEYS;
      const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
      const unsigned s_addr = tmem_s + lanes + (unsigned)(g * 64 + first_key), o_addr = tmem_o + lanes + (unsigned)(g * S::OUT);
      unsigned char* p_row = p_s + g * P_BYTES + r * 128;
      const bool real = row < p.rows;
      const int token = real ? (p.row0 + row) / per_kv - p.row0 / per_kv : -2;
      const int high = real ? p.position[token] : -1, low = real ? p.low[token] : 0;
      const float scale = a.scale * 1.4426950408889634f;
      float m_run = -INFINITY, l_run = 0.f;
      bool ok = true;
      int taken = 0;
      // (a wait that ran out is not left at once: the warps of a group meet at barriers that they all have to reach)
      for (int j = g; j < steps; j += GROUPS, ++taken) {
        int whose;
        const int at = look_up(p, begin + j, whose) * PAGE;
        const bool edge = whose >= 0 || at < p.all_from || at + PAGE - 1 > p.all_to;
        ok = ok && mbar_wait(&bar.s_full[g], (j / GROUPS) & 1);
        __syncwarp();
        fence_after_sync();
        float v[KEYS];
#pragma unroll
        for (int c = 0; c < KEYS; c += 16) tmem_load16_nowait(s_addr + (unsigned)c, reinterpret_cast<unsigned*>(v) + c);
        tmem_wait_ld();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.s_empty[g]);
#pragma unroll
        for (int c = 0; c < KEYS; ++c) v[c] *= scale;
        unsigned long long seen = ~0ull;
        if (edge) {
          const bool mine = whose < 0 || whose == token;
          seen = 0ull;
#pragma unroll
          for (int c = 0; c < KEYS; ++c) {
            const int key = at + first_key + c;
            const bool sees = mine && key <= high && key >= low;
            if (sees) seen |= 1ull << c;
            else v[c] = -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < KEYS; ++c) mx[c & 3] = fmaxf(mx[c & 3], v[c]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        float fade = 1.f;
        if (top > m_run + 8.f) {  // (also a row's first scores, while its maximum is still -inf)
          fade = fast_exp2(m_run - top);
          m_run = top;
        }
        const float shift = m_run > -INFINITY ? m_run : 0.f;
        unsigned packed[KEYS / 2];
#pragma unroll
        for (int c = 0; c < KEYS; c += 2) {
          const float w0 = fast_exp2(v[c] - shift), w1 = fast_exp2(v[c + 1] - shift);
          sum[c & 3] += w0;
          sum[(c + 1) & 3] += w1;
          packed[c / 2] = pack_bf16(w0, w1);
        }
        l_run = l_run * fade + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        // the group's previous product has to be over: it reads P and adds to the outputs
        if (taken >= 1) {
          ok = ok && mbar_wait(&bar.o_full[g], ((j - GROUPS) / GROUPS) & 1);
          __syncwarp();
          fence_after_sync();
        }
#pragma unroll
        for (int c = 0; c < KEYS / 8; ++c)
          *reinterpret_cast<uint4*>(p_row + (((first_key / 8 + c) ^ (r & 7)) << 4)) =
              make_uint4(packed[4 * c], packed[4 * c + 1], packed[4 * c + 2], packed[4 * c + 3]);
        bool odd = false;
        const unsigned char* v_tile = v_s + (j % V_STAGES) * KV_BYTES;
        if (edge) {
          ok = ok && mbar_wait(&bar.v_full[j % V_STAGES], (j / V_STAGES) & 1);
#pragma unroll
          for (int i = 0; i < KV_BYTES / 16 / 128; ++i) {
            uint4 x = *reinterpret_cast<const uint4*>(v_tile + (i * 128 + r) * 16);
            odd = odd || odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w);
          }
          if (__any_sync(0xffffffffu, odd) && lane == 0) odd_s[g] = 1;
          asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory");
          odd = *(volatile int*)&odd_s[g] != 0;
          asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory");
          if (r == 0) { odd_s[g] = 0; *(volatile int*)&skip_s[g] = odd; }
        } else if (r == 0) {
          *(volatile int*)&skip_s[g] = 0;
        }
        if (odd || (taken >= 1 && __any_sync(0xffffffffu, fade != 1.f))) {
#pragma unroll 1
          for (int c = 0; c < S::OUT; c += 16) {
            unsigned o[16];
            if (taken >= 1) tmem_load16(o_addr + (unsigned)c, o);
#pragma unroll
            for (int d = 0; d < 16; ++d) o[d] = taken >= 1 ? __float_as_uint(__uint_as_float(o[d]) * fade) : 0u;
            if (odd) {
#pragma unroll 1
              for (int key = 0; key < KEYS; ++key) {
                if (!(seen >> key & 1ull)) continue;
                const int at_key = first_key + key;
                const float w = __bfloat162float(*reinterpret_cast<const bf16*>(p_row + (((at_key >> 3) ^ (r & 7)) << 4) + 2 * (at_key & 7)));
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                  const int column = (c & 63) + d;
                  const bf16 x = *reinterpret_cast<const bf16*>(v_tile + (c >> 6) * 8192 + at_key * 128 + (((column >> 3) ^ (at_key & 7)) << 4) + 2 * (column & 7));
                  o[d] = __float_as_uint(fmaf(w, __bfloat162float(x), __uint_as_float(o[d])));
                }
              }
              __syncwarp();
            }
            tmem_store16(o_addr + (unsigned)c, o);
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
      // ---- groups and copies together: a common maximum, then sums through shared memory (P and the stages are free: every
      // product has been added)
      sm_m[g][r] = m_run;
      sm_l[g][r] = l_run;
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i)
#pragma unroll
        for (int copy = 0; copy < COPIES; ++copy) top = fmaxf(top, sm_m[i][copy * ROWS + row]);
      const float w = m_run > -INFINITY ? fast_exp2(m_run - top) : 0.f;
      float* ex = reinterpret_cast<float*>(p_s);
#pragma unroll 1
      for (int c = 0; c < S::OUT; c += 16) {
        unsigned o[16];
        if (taken >= 1) tmem_load16(o_addr + (unsigned)c, o);
#pragma unroll
        for (int d = 0; d < 16; d += 4) {
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (taken >= 1 && w != 0.f)
            x = make_float4(__uint_as_float(o[d]) * w, __uint_as_float(o[d + 1]) * w, __uint_as_float(o[d + 2]) * w, __uint_as_float(o[d + 3]) * w);
          *reinterpret_cast<float4*>(ex + (size_t)(g * 128 + r) * S::LD + c + d) = x;
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      const int fours = hd / 4;
      for (int i = tid; i < p.rows * fours; i += SOFT_WARPS * 32) {
        const int to = i / fours, d = (i % fours) * 4;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        float most = -INFINITY, total = 0.f;
#pragma unroll
        for (int e = 0; e < GROUPS * COPIES; ++e) most = fmaxf(most, sm_m[e / COPIES][e % COPIES * ROWS + to]);
#pragma unroll
        for (int e = 0; e < GROUPS * COPIES; ++e) {
          const int from = e % COPIES * ROWS + to;
          float4 y = *reinterpret_cast<const float4*>(ex + (size_t)(e / COPIES * 128 + from) * S::LD + d);
          x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
          const float me = sm_m[e / COPIES][from], le = sm_l[e / COPIES][from];
          total += me > -INFINITY ? le * fast_exp2(me - most) : le;
        }
        if (a.splits == 1) {
          const float inv = total != 0.f ? 1.f / total : 0.f;
          const int in_group = p.row0 + to, t = p.token0 + in_group / per_kv - p.row0 / per_kv;
          *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + ((size_t)t * a.heads + kv * per_kv + in_group % per_kv) * hd + d) =
              make_uint2(pack_bf16(x.x * inv, x.y * inv), pack_bf16(x.z * inv, x.w * inv));
        } else {
          *reinterpret_cast<float4*>(a.scratch + ((pair * a.splits + blockIdx.x) * ROWS + to) * hd + d) = x;
          if (d == 0) {
            float* ml = a.scratch + (size_t)gridDim.z * gridDim.y * a.splits * ROWS * hd + ((pair * a.splits + blockIdx.x) * ROWS + to) * 2;
            *reinterpret_cast<float2*>(ml) = make_float2(most, total);
          }
        }
      }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == SOFT_WARPS + 1) tmem_dealloc(tmem_base_s, S::COLUMNS);
  }
  if (a.splits == 1) return;
  if (is_last(p, a, pair)) join<bf16, ROWS, THREADS>(p, a, pair, reinterpret_cast<float*>(tiles));
}

template <int BOXES, int COPIES>
int launch(const Args& a, long long pages, dim3 grid, cudaStream_t stream) {
  typedef Shape<BOXES> S;
  static_assert((MAX_SPLITS + 1) * 128 * 4 + 1024 <= S::SMEM, "the weights of the join");
  CUtensorMap map;
  if (!make_map(&map, a.cache.base, pages * 2 * a.cache.kv_heads * PAGE, a.cache.head_dim, PAGE)) return DLLM_LAUNCH_FAILED;
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)kernel<BOXES, COPIES>, S::SMEM, done)) return DLLM_LAUNCH_FAILED;
  return dllm_launch_pdl(kernel<BOXES, COPIES>, grid, dim3(THREADS), S::SMEM, stream, map, a);
}
}  // namespace t5

// ---- everything else ---------------------------------------------------------------------------------------------
// 16 query rows a tile, 128 threads. A page's keys, then its values, lie in shared memory as float32. Scores: a thread has one
// key and half of the rows; the softmax: a warp four rows; the sums: a thread four dimensions and some of the rows.
constexpr int FMA_ROWS = 16, FMA_THREADS = 128, FMA_DIM = 256;

template <typename T>
__global__ void __launch_bounds__(FMA_THREADS) fma_kernel(const Args a) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ Plan p;
  __shared__ float sm_p[FMA_ROWS][PAGE + 1], sm_m[FMA_ROWS], sm_l[FMA_ROWS], sm_fade[FMA_ROWS];
  __shared__ int row_token[FMA_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = a.cache.head_dim, kv = blockIdx.y, per_kv = a.heads / a.cache.kv_heads, ld = hd + 4;
  float* q_s = reinterpret_cast<float*>(smem_raw);  // [FMA_ROWS][ld]
  float* tile = q_s + FMA_ROWS * ld;                 // [PAGE][ld]
  pdl_launch_dependents();
  pdl_wait();
  make_plan(p, a, FMA_ROWS);
  if (p.rows == 0) return;
  const size_t pair = (size_t)blockIdx.z * gridDim.y + kv;
  const int begin = (int)((long long)p.total * blockIdx.x / a.splits), end = (int)((long long)p.total * (blockIdx.x + 1) / a.splits);
  const int fours = hd / 4;
  if (begin < end || a.splits == 1) {
    for (int i = tid; i < FMA_ROWS * hd; i += FMA_THREADS) {
      int r = i / hd, d = i % hd, row = p.row0 + r;
      float v = 0.f;
      if (r < p.rows)
        v = to_float(static_cast<const T*>(a.q)[((size_t)(p.token0 + row / per_kv - p.row0 / per_kv) * a.heads + kv * per_kv + row % per_kv) * hd + d]);
      q_s[r * ld + d] = v;
    }
    if (tid < FMA_ROWS) {
      sm_m[tid] = -INFINITY;
      sm_l[tid] = 0.f;
      row_token[tid] = tid < p.rows ? (p.row0 + tid) / per_kv - p.row0 / per_kv : -2;
    }
    // sums: this thread's four dimensions (of up to 64) and rows: tid / fours, then in steps
    const int columns = min(fours, FMA_THREADS), step = FMA_THREADS / columns;
    const int d4 = (tid % columns) * 4, r_first = tid / columns;
    const bool sums = r_first < step;
    float4 acc[FMA_ROWS];  // (rows r_first + step * i)
#pragma unroll
    for (int i = 0; i < FMA_ROWS; ++i) acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float scale = a.scale * 1.4426950408889634f;
    const T* base = static_cast<const T*>(a.cache.base);
    __syncthreads();
    for (int part = begin; part < end; part += LIST) {
      const int count = min(LIST, end - part);
      list_pages(p, a, part, part + count);
      for (int it = 0; it < count; ++it) {
        const int whose = p.whose[it], at = p.at[it];
        auto fetch = [&](int which) {
          const T* src = base + kv_offset(a.cache, p.page[it], which, kv, 0);
          int from = whose < 0 ? 0 : p.low[whose], to = whose < 0 ? p.position[p.longest] : p.position[whose];
          for (int i = tid; i < PAGE * fours; i += FMA_THREADS) {
            int r = i / fours, d = (i % fours) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at + r >= from && at + r <= to) {
              const T* s = src + (size_t)r * hd + d;
              v = make_float4(to_float(s[0]), to_float(s[1]), to_float(s[2]), to_float(s[3]));
            }
            *reinterpret_cast<float4*>(tile + r * ld + d) = v;
          }
        };
        fetch(0);
        __syncthreads();
        {
          const int key = tid & 63, half = tid >> 6;
          float dot[FMA_ROWS / 2];
#pragma unroll
          for (int i = 0; i < FMA_ROWS / 2; ++i) dot[i] = 0.f;
          for (int d = 0; d < hd; d += 4) {
            float4 k4 = *reinterpret_cast<const float4*>(tile + key * ld + d);
#pragma unroll
            for (int i = 0; i < FMA_ROWS / 2; ++i) {
              float4 q4 = *reinterpret_cast<const float4*>(q_s + (half * (FMA_ROWS / 2) + i) * ld + d);
              dot[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, dot[i]))));
            }
          }
#pragma unroll
          for (int i = 0; i < FMA_ROWS / 2; ++i) {
            int r = half * (FMA_ROWS / 2) + i, t = row_token[r];
            bool sees = t >= 0 && (whose < 0 || whose == t) && at + key <= p.position[t] && at + key >= p.low[t];
            sm_p[r][key] = sees ? dot[i] * scale : -INFINITY;
          }
        }
        __syncthreads();
        fetch(1);
        for (int r = warp; r < FMA_ROWS; r += FMA_THREADS / 32) {
          float x0 = sm_p[r][lane], x1 = sm_p[r][lane + 32];
          float top = fmaxf(warp_max(fmaxf(x0, x1)), sm_m[r]);
          float shift = top > -INFINITY ? top : 0.f;
          // (a masked key's weight is marked by -1: its value is not multiplied)
          float w0 = x0 == -INFINITY ? 0.f : exp2f(x0 - shift), w1 = x1 == -INFINITY ? 0.f : exp2f(x1 - shift);
          float sum = warp_sum(w0 + w1);
          sm_p[r][lane] = x0 == -INFINITY ? -1.f : w0;
          sm_p[r][lane + 32] = x1 == -INFINITY ? -1.f : w1;
          if (lane == 0) {
            float fade = sm_m[r] > -INFINITY ? exp2f(sm_m[r] - shift) : 0.f;
            sm_fade[r] = fade;
            sm_l[r] = sm_l[r] * fade + sum;
            sm_m[r] = top;
          }
        }
        __syncthreads();
        if (sums) {
#pragma unroll
          for (int i = 0; i < FMA_ROWS; ++i) {
            int r = r_first + step * i;
            if (r < FMA_ROWS) {
              float f = sm_fade[r];
              acc[i].x *= f; acc[i].y *= f; acc[i].z *= f; acc[i].w *= f;
            }
          }
          for (int key = 0; key < PAGE; ++key) {
            float4 v = *reinterpret_cast<const float4*>(tile + key * ld + d4);
#pragma unroll
            for (int i = 0; i < FMA_ROWS; ++i) {
              int r = r_first + step * i;
              if (r < FMA_ROWS) {
                float w = sm_p[r][key];
                if (w != -1.f) {
                  acc[i].x = fmaf(w, v.x, acc[i].x);
                  acc[i].y = fmaf(w, v.y, acc[i].y);
                  acc[i].z = fmaf(w, v.z, acc[i].z);
                  acc[i].w = fmaf(w, v.w, acc[i].w);
                }
              }
            }
          }
        }
        __syncthreads();
      }
    }
    if (sums) {
#pragma unroll
      for (int i = 0; i < FMA_ROWS; ++i) {
        int r = r_first + step * i;
        if (r < FMA_ROWS && r < p.rows) {
          if (a.splits == 1) {
            float inv = sm_l[r] != 0.f ? 1.f / sm_l[r] : 0.f;
            int row = p.row0 + r, t = p.token0 + row_token[r];
            T* to = static_cast<T*>(a.out) + ((size_t)t * a.heads + kv * per_kv + row % per_kv) * hd + d4;
            to[0] = from_float<T>(acc[i].x * inv);
            to[1] = from_float<T>(acc[i].y * inv);
            to[2] = from_float<T>(acc[i].z * inv);
            to[3] = from_float<T>(acc[i].w * inv);
          } else {
            *reinterpret_cast<float4*>(a.scratch + ((pair * a.splits + blockIdx.x) * FMA_ROWS + r) * hd + d4) = acc[i];
          }
        }
      }
    }
    if (a.splits > 1 && tid < p.rows) {
      float* ml = a.scratch + (size_t)gridDim.z * gridDim.y * a.splits * FMA_ROWS * hd + ((pair * a.splits + blockIdx.x) * FMA_ROWS + tid) * 2;
      *reinterpret_cast<float2*>(ml) = make_float2(sm_m[tid], sm_l[tid]);
    }
  }
  if (a.splits == 1) return;
  if (is_last(p, a, pair)) join<T, FMA_ROWS, FMA_THREADS>(p, a, pair, reinterpret_cast<float*>(smem_raw));
}

// ---- launch shapes -------------------------------------------------------------------------------------------------
enum { FMA = 0, MMA = 1, TCGEN05 = 2 };
struct Shape { int kind, rows, tiles, splits; };

// `kind`: -1 chooses.
Shape shape_of(int kind, int dtype, int heads, int kv_heads, int head_dim, int groups, int max_rows, int max_context) {
  Shape s;
  const int query_rows = max_rows * (heads / kv_heads);
  const bool mma = dtype == DLLM_BF16 && head_dim % 16 == 0 && head_dim <= 128, tcgen05 = mma && head_dim >= 64;
  const int pages = (max_context + PAGE - 1) / PAGE;
  s.kind = kind >= 0 ? kind : tcgen05 && pages > 4 ? TCGEN05 : mma ? MMA : FMA;
  if ((s.kind == TCGEN05 && !tcgen05) || (s.kind == MMA && !mma)) s.kind = FMA;
  if (s.kind == FMA) s.rows = FMA_ROWS;
  else if (s.kind == MMA) s.rows = query_rows <= 16 ? 16 : query_rows <= 32 ? 32 : 64;
  else s.rows = query_rows <= 32 ? 32 : query_rows <= 64 ? 64 : 128;
  s.tiles = (query_rows + s.rows - 1) / s.rows;
  // as many splits as the device has places for, but not more than there can be pages
  const long long pairs = (long long)groups * s.tiles * kv_heads;
  const long long places = 148LL * (s.kind == TCGEN05 && head_dim > 64 ? 1 : 2);
  long long splits = places / (pairs > 0 ? pairs : 1);
  if (splits > pages + max_rows) splits = pages + max_rows;
  if (splits > MAX_SPLITS) splits = MAX_SPLITS;
  s.splits = splits < 1 ? 1 : (int)splits;
  return s;
}

template <int HD, int MT, int WM, int STAGES>
int launch_mma(const Args& a, dim3 grid, cudaStream_t stream) {
  constexpr int ROWS = 16 * MT * WM;
  constexpr int ring = STAGES * 2 * 64 * HD * 2, sums = 4 * ROWS * HD * 4;
  constexpr int weights = (MAX_SPLITS + 1) * ROWS * 4;
  constexpr int bytes = ROWS * HD * 2 + (ring > sums ? ring : sums);
  constexpr int smem = bytes > weights ? bytes : weights;
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)mma_kernel<HD, MT, WM, STAGES>, smem, done)) return DLLM_LAUNCH_FAILED;
  return dllm_launch_pdl(mma_kernel<HD, MT, WM, STAGES>, grid, dim3(WM * 128), smem, stream, a);
}

template <typename T>
int launch_fma(const Args& a, dim3 grid, cudaStream_t stream) {
  const int tiles = (FMA_ROWS + PAGE) * (a.cache.head_dim + 4) * 4, weights = (a.splits + 1) * FMA_ROWS * 4;
  static std::atomic<unsigned long long> done{0};
  if (!dllm_allow_shared((const void*)fma_kernel<T>, (FMA_ROWS + PAGE) * (FMA_DIM + 4) * 4, done)) return DLLM_LAUNCH_FAILED;
  return dllm_launch_pdl(fma_kernel<T>, grid, dim3(FMA_THREADS), tiles > weights ? tiles : weights, stream, a);
}
}  // namespace

// Query rows of a tile in the low 16 bits, splits above: scratch holds groups x tiles x kv_heads x splits x rows x
// (head_dim + 2) floats, tickets groups x tiles x kv_heads words. kind: -1, or 0, 1, 2 (fused multiply-adds, mma.sync, tcgen05).
DLLM_EXPORT int dllm_attention_shared_shape(int kind, int dtype, int heads, int kv_heads, int head_dim, int groups, int max_rows,
                                            int max_context) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || groups <= 0 || max_rows <= 0 || max_context <= 0) return DLLM_BAD_ARGUMENT;
  Shape s = shape_of(kind, dtype, heads, kv_heads, head_dim, groups, max_rows, max_context);
  return s.rows | s.splits << 16;
}

// See the head of the file. out, q [tokens, heads * head_dim] in the cache's type; slots, positions: each token's table row and
// position; cuts [groups + 1]: the groups' first tokens; shared [groups]: pages from the first on that a group's table rows have
// in common; the cache entry has `pages` pages.
DLLM_EXPORT int dllm_attention_shared(int kind, void* out, const void* q, void* base, long long pages, const int* page_table,
                                      int max_pages, int page_size, int dtype, int heads, int kv_heads, int head_dim,
                                      const int* slots, const int* positions, const int* cuts, const int* shared, int groups,
                                      int max_rows, int max_context, float scale, int window, float* scratch, unsigned* tickets,
                                      int* status, cudaStream_t stream) {
  if (groups <= 0 || max_rows <= 0) return DLLM_OK;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_context <= 0 || window < 0 || pages <= 0) return DLLM_BAD_ARGUMENT;
  if (head_dim % 8 || head_dim <= 0 || head_dim > FMA_DIM || page_size != PAGE || kv_heads > 65535 ||
      ((uintptr_t)out | (uintptr_t)q | (uintptr_t)base) & 15)
    return DLLM_UNSUPPORTED_SIZE;
  Shape s = shape_of(kind, dtype, heads, kv_heads, head_dim, groups, max_rows, max_context);
  if ((long long)groups * s.tiles > 65535) return DLLM_UNSUPPORTED_SIZE;
  Args a{out, q, KvLayout{base, page_table, max_pages, page_size, kv_heads, head_dim}, slots, positions, cuts, shared, scratch,
         tickets, status, heads, window, s.tiles, s.splits, scale};
  dim3 grid(s.splits, kv_heads, groups * s.tiles);
  if (s.kind == FMA) return dtype == DLLM_BF16 ? launch_fma<bf16>(a, grid, stream) : launch_fma<float>(a, grid, stream);
  if (s.kind == TCGEN05) {
    if (pages * 2 * kv_heads * PAGE > 0x7fffffffll) return DLLM_UNSUPPORTED_SIZE;
    if (head_dim <= 64) {
      if (s.rows == 32) return t5::launch<1, 4>(a, pages, grid, stream);
      if (s.rows == 64) return t5::launch<1, 2>(a, pages, grid, stream);
      return t5::launch<1, 1>(a, pages, grid, stream);
    }
    if (s.rows == 32) return t5::launch<2, 4>(a, pages, grid, stream);
    if (s.rows == 64) return t5::launch<2, 2>(a, pages, grid, stream);
    return t5::launch<2, 1>(a, pages, grid, stream);
  }
  if (head_dim <= 32) {
    if (s.rows == 16) return launch_mma<32, 1, 1, 4>(a, grid, stream);
    if (s.rows == 32) return launch_mma<32, 2, 1, 4>(a, grid, stream);
    return launch_mma<32, 2, 2, 4>(a, grid, stream);
  }
  if (head_dim <= 64) {
    if (s.rows == 16) return launch_mma<64, 1, 1, 4>(a, grid, stream);
    if (s.rows == 32) return launch_mma<64, 2, 1, 4>(a, grid, stream);
    return launch_mma<64, 2, 2, 4>(a, grid, stream);
  }
  if (s.rows == 16) return launch_mma<128, 1, 1, 3>(a, grid, stream);
  if (s.rows == 32) return launch_mma<128, 2, 1, 3>(a, grid, stream);
  return launch_mma<128, 2, 2, 4>(a, grid, stream);
}
