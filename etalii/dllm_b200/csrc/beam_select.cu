// The choice of beam search: from the logits of every beam of a sequence and the beams' scores to the next beams, and the
// pool of texts that ended.
//
// A row x of logits (float32) is a beam's; lse = m + log(sum exp(x - m)), m its maximum. The candidate that continues
// beam k with token t has total (x_t - lse) + score_k. Candidates are ordered by total, then by beam (ascending), then by
// logit, then by token (ascending): within a row that is the order of the logits, so a row's best candidates are known
// before its lse is. Only totals above -inf count (a row of which nothing is left, or that holds a NaN or +inf, has none).
//   next beams: the best `beams` candidates that are no stop tokens. A beam's first continuation keeps the beam's place, the
//     others take the free places in order: what moves between places then moves as little as it can.
//   ended texts: stop tokens among the first `beams` of all candidates enter the sequence's pool (kept in descending order,
//     at most `beams` long, earlier entries first among equals) at total / (produced + 1)^penalty.
//   done: the pool is full and (early, or its last is no worse than the best live total / (produced + 1)^penalty), or no
//     beam lives. A sequence that is done keeps its pool, and its places get score -inf.
//
// One pass over the logits, in two steps of one launch:
//   1. A block walks a stretch of a row in tiles of 256 threads x 4 * REG logits, a thread with a maximum and a sum of its own.
//      Lane i of all warps is group i; the beams-th largest of the 32 groups' maxima so far is a bound that at least `beams`
//      logits reach and few do: of logits in any order 4.3, 9.2, 22 for 4, 8, 16 beams (32 H(32) = 130 for 32), so that looking for
//      them costs little: with the smallest maximum of as many groups as beams or more as the bound, 54 of them for 16
//      groups, most of the instructions were theirs (32 x 16 beams on 128,256 logits 60.7 us, now 55.4; 1 x 4 on 49,152 9.7, now
//      8.3). What of a tile reaches the bound goes to a list, which is thinned out by the latest bound when it fills; at the end each entry counts
//      what is before it. A list that does not hold them all (many equal logits) is given up for `beams` passes over the stretch.
//   2. The block that finishes last for its sequence (a ticket counter; nobody waits) joins the stretches' sums,
//      makes the totals and chooses among the stretches' lists the same way; a warp deals out places and pool.
// Bound by HBM where the rows are many, by the latency of the two steps where they are few: 1 x 4 beams of 49,152 logits 8.1 us (2.5 to the
// stretch's best, 1 for the ticket, 4 for the join), 8 x 8 of 128,256 18.5, 32 x 16 54.9 (230 MB of living rows, 4.2 TB/s; 6.3 while all
// multiprocessors have as many blocks, but 448 living rows are four for some and three for others). Blocks of a stretch that fits
// their registers (4,096 of them for 512 rows of 128,256 instead of 512) spent most of their time on what a block costs. The next tile
// by bulk copies into shared memory while this one is worked on changed nothing (8 x 8 18.0 us where it was 18.7, 32 x 16 57.1 where it was 55.4).
#include <float.h>

#include "common.cuh"

namespace {
constexpr int THREADS = 256;
constexpr int MAX_BEAMS = 32, MAX_STOPS = 8;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int LIST = 1024;       // candidates a block keeps
constexpr int PLACES = 148 * 4;  // blocks that are resident at a time

struct Args {
  const float* logits;
  long long row_stride;
  const float *scores, *finished;
  const int *finished_at, *done, *produced, *steps, *stop_ids;
  float *scores_out, *finished_out;
  int *finished_at_out, *done_out, *parents, *tokens, *history;
  float* scratch;                // [row][stretch]: maximum, sum, then `beams` pairs (logit, token)
  unsigned* tickets;             // one a sequence, zero between launches
  int beams_in, beams, vocab, n_stops, min_tokens, early, stretch, history_steps;
  float penalty;
};

// (total, beam, logit, token) in the order of the choice
struct Candidate {
  float total, logit;
  int beam, token;
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  if (a.total != b.total) return a.total > b.total;
  if (a.beam != b.beam) return a.beam < b.beam;
  if (a.logit != b.logit) return a.logit > b.logit;
  return a.token < b.token;
}

struct Shared {
  // a stretch's candidates as words that order them (`word_of`); a sequence's as logit and token, total, beam
  unsigned long long list[LIST], kept[LIST];
  float list_total[LIST];
  int list_beam[LIST];
  float lane_max[2][THREADS / 32][32];
  float warp_m[THREADS / 32], warp_f[THREADS / 32];
  int list_n, seen_n[2], kept_n, last;
  unsigned long long best[2];
  float lse[MAX_BEAMS], score[MAX_BEAMS];
  Candidate chosen[MAX_BEAMS];
  Candidate stop[MAX_BEAMS * MAX_STOPS];
  float chosen_total[MAX_BEAMS], stop_total[MAX_BEAMS * MAX_STOPS];
  Candidate ended[MAX_BEAMS];
  int n_ended;
  int stops[MAX_STOPS];
};

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

__device__ __forceinline__ unsigned ordered(float v) {  // larger floats have larger words; no NaN comes here
  unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Orders a row's candidates: by logit, then by the lower token.
__device__ __forceinline__ unsigned long long word_of(float logit, int token) {
  return ((unsigned long long)ordered(logit) << 32) | (unsigned)(0x7fffffff - token);
}
__device__ __forceinline__ float logit_of(unsigned long long word) {
  const unsigned w = (unsigned)(word >> 32);
  return __uint_as_float(w & 0x80000000u ? w & 0x7fffffffu : ~w);
}
__device__ __forceinline__ int token_of(unsigned long long word) { return 0x7fffffff - (int)(unsigned)word; }

// The rank-th largest of the lanes' maxima of v over the warps, which every thread gets. (A short stretch has something of
// every lane.) `set`: 0 and 1 in turn.
__device__ __forceinline__ float bound_of(float v, int rank, Shared& sh, int set) {
  const int lane = threadIdx.x & 31;
  sh.lane_max[set][threadIdx.x >> 5][lane] = v;
  __syncthreads();
  v = -INFINITY;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v = fmaxf(v, sh.lane_max[set][w][lane]);
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)  // sorts the lanes' values, the largest first: lane i holds the i-th
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) {
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      const bool first = (lane & o) == 0, down = (lane & size) == 0;
      v = first == down ? fmaxf(v, other) : fminf(v, other);
    }
  return __shfl_sync(0xffffffffu, v, rank - 1);
}

// What is done and what its places hold from then on.
__device__ __forceinline__ void leave_as_is(const Args& a, int b, int* history) {
  for (int i = threadIdx.x; i < a.beams; i += THREADS) {
    size_t at = (size_t)b * a.beams + i;
    a.scores_out[at] = -INFINITY;
    a.parents[at] = min(i, a.beams_in - 1);
    if (history) history[i] = min(i, a.beams_in - 1);
    a.tokens[at] = 0;
    if (a.finished_out != a.finished) a.finished_out[at] = a.finished[at];
    if (a.finished_at_out != a.finished_at) {
      a.finished_at_out[2 * at] = a.finished_at[2 * at];
      a.finished_at_out[2 * at + 1] = a.finished_at[2 * at + 1];
    }
  }
  if (threadIdx.x == 0) a.done_out[b] = 1;
}

template <int REG>
__global__ void __launch_bounds__(THREADS, 4) select_kernel(const Args a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, b = row / a.beams_in, k = row % a.beams_in;
  const int part = blockIdx.x, parts = gridDim.x;
  const int beams = a.beams, vocab = a.vocab;
  if (tid == 0) sh.list_n = sh.kept_n = sh.n_ended = sh.seen_n[0] = sh.seen_n[1] = 0;
  pdl_launch_dependents();
  pdl_wait();
  // ---- the stretch: whole fours where addresses are multiples of 16 bytes; the up to three logits before and behind those are
  // `extra` of threads 0 to 2 and 4 to 6. The first tile is asked for before anything is looked at.
  const float* x = a.logits + (size_t)row * a.row_stride;
  const int lo = min(vocab, part * a.stretch), hi = min(vocab, lo + a.stretch);
  const int first = min(hi, lo + (int)((0 - (reinterpret_cast<uintptr_t>(x + lo) >> 2)) & 3));
  const int fours = (hi - first) >> 2, behind = first + 4 * fours;
  const float4* x4 = reinterpret_cast<const float4*>(x + first);
  float v[4 * REG];
  auto load = [&](int tile) {
    const int at0 = tile * REG * THREADS + tid;
    if ((tile + 1) * REG * THREADS <= fours) {
#pragma unroll
      for (int r = 0; r < REG; ++r) {
        const float4 four = __ldcs(x4 + at0 + r * THREADS);
        v[4 * r] = four.x; v[4 * r + 1] = four.y; v[4 * r + 2] = four.z; v[4 * r + 3] = four.w;
      }
    } else {
#pragma unroll
      for (int r = 0; r < REG; ++r) {
        float4 four = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at0 + r * THREADS < fours) four = __ldcs(x4 + at0 + r * THREADS);
        v[4 * r] = four.x; v[4 * r + 1] = four.y; v[4 * r + 2] = four.z; v[4 * r + 3] = four.w;
      }
    }
  };
  load(0);
  int extra_at = -2;
  if (tid < 3 && lo + tid < first) extra_at = lo + tid;
  if (tid >= 4 && tid < 7 && behind + tid - 4 < hi) extra_at = behind + tid - 4;
  const float extra = extra_at >= 0 ? __ldcs(x + extra_at) : -INFINITY;
  const int run_step = a.steps ? a.steps[0] : 0, step = a.produced[0] + run_step, sequences = gridDim.y / a.beams_in;
  const bool over = a.done[b] != 0, alive = a.scores[(size_t)b * a.beams_in + k] > -INFINITY;
  if (tid < a.n_stops) sh.stops[tid] = a.stop_ids[tid];
  // where the parents of this step are kept too
  int* history = a.history && run_step < a.history_steps ? a.history + ((size_t)run_step * sequences + b) * beams : nullptr;
  if (over) {
    if (k == 0 && part == 0) leave_as_is(a, b, history);
    return;
  }
  __syncthreads();
  const int n_stops = a.n_stops;
  auto is_stop = [&](int i) {
    bool stop = false;
    for (int s = 0; s < n_stops; ++s) stop = stop || sh.stops[s] == i;
    return stop;
  };
  float* mine = a.scratch + ((size_t)row * parts + part) * (2 + 2 * beams);
  if (alive) {
    auto place_of = [&](int tile, int e) { return first + 4 * ((tile * REG + (e >> 2)) * THREADS + tid) + (e & 3); };
    auto offer = [&](float value, int i) {
      if (is_stop(i)) return;
      int at = atomicAdd(&sh.list_n, 1);
      if (at < LIST) sh.list[at] = word_of(value, i);
    };
    float m = extra, sum = extra > -INFINITY ? 1.f : 0.f, keep = -INFINITY, low = -INFINITY;
    if (extra != extra) sum = extra;  // (a NaN is the row's end)
    if (extra_at >= 0 && !is_stop(extra_at)) keep = extra;
    float floor_ = -FLT_MAX;
    int updates = 0;
    const int tiles = max(1, (fours + REG * THREADS - 1) / (REG * THREADS));
    for (int tile = 0; tile < tiles; ++tile) {
      if (tile > 0) load(tile);
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4 * REG; ++e) top = fmaxf(top, v[e]);
      // The bound goes by what may be chosen: what a thread has in a tile beside a stop token does not take part in it (any
      // logits of at least `beams` lanes make a bound).
      bool beside = false;
      for (int s = 0; s < n_stops; ++s) {
        const int at = ((sh.stops[s] - first) >> 2) - tile * REG * THREADS;
        beside = beside || (sh.stops[s] >= first && sh.stops[s] < behind && at >= 0 && at < REG * THREADS && at % THREADS == tid);
      }
      if (!beside) keep = fmaxf(keep, top);
      if ((tile & (tile - 1)) == 0) {  // a new bound with the first, the second, the third, the fifth, the ninth tile ..: no barrier between
        if (tid == 0) sh.seen_n[updates & 1] = sh.list_n;  // (of the tiles before; a late entry of the last one may be missing)
        low = bound_of(keep, beams, sh, updates & 1);
        floor_ = fmaxf(low, -FLT_MAX);  // (-inf is no candidate)
        if (sh.seen_n[updates & 1] > LIST / 2) {  // thin out the list
          __syncthreads();
          const int n = min(sh.list_n, LIST);
          unsigned long long kept[LIST / THREADS];
#pragma unroll
          for (int u = 0; u < LIST / THREADS; ++u) kept[u] = u * THREADS + tid < n ? sh.list[u * THREADS + tid] : 0ull;
          const bool lost = sh.list_n > LIST;
          __syncthreads();
          if (tid == 0) sh.list_n = lost ? LIST + 1 : 0;  // (what is lost stays lost)
          __syncthreads();
          if (!lost)
#pragma unroll
            for (int u = 0; u < LIST / THREADS; ++u)
              if (kept[u] >= word_of(floor_, 0x7fffffff)) sh.list[atomicAdd(&sh.list_n, 1)] = kept[u];
          __syncthreads();
        }
        ++updates;
      }
      const float m_new = fmaxf(m, top), shift = m_new > -INFINITY ? -m_new : 0.f;
      Two sums[2] = {two(0.f, 0.f), two(0.f, 0.f)};
      const Two shift2 = two(shift, shift), log2e2 = two(LOG2E, LOG2E);
#pragma unroll
      for (int e = 0; e < 4 * REG; e += 2) {  // (the difference first: it is exact where the weight is large)
        const float2 y = apart(mul2(add2(two(v[e], v[e + 1]), shift2), log2e2));
        sums[e >> 1 & 1] = add2(sums[e >> 1 & 1], two(fast_exp2(y.x), fast_exp2(y.y)));
      }
      const float2 all_four = apart(add2(sums[0], sums[1]));
      sum = sum * (m > -INFINITY ? fast_exp2((m + shift) * LOG2E) : 1.f) + (all_four.x + all_four.y);
      m = m_new;
      if (top >= floor_) {  // (few threads of a tile have something that reaches the bound)
        unsigned hits = 0u;
#pragma unroll
        for (int e = 0; e < 4 * REG; ++e) hits |= v[e] >= floor_ ? 1u << e : 0u;
        while (hits) {
          const int e = __ffs(hits) - 1;
          hits &= hits - 1;
          float value = v[0];
#pragma unroll
          for (int j = 1; j < 4 * REG; ++j) value = e == j ? v[j] : value;
          offer(value, place_of(tile, e));
        }
      }
    }
    if (extra >= fmaxf(low, -FLT_MAX)) offer(extra, extra_at);
    // ---- the stretch's maximum and sum, its best
    const float warp_top = warp_max(m);
    sum = warp_sum(m > -INFINITY ? sum * fast_exp2((m - warp_top) * LOG2E) : sum);  // (0 where there is nothing, or a NaN)
    if (lane == 0) { sh.warp_m[warp] = warp_top; sh.warp_f[warp] = sum; }
    __syncthreads();
    if (tid == 0) {
      float top = -INFINITY, total = 0.f;
      for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, sh.warp_m[w]);
      for (int w = 0; w < THREADS / 32; ++w)
        total += sh.warp_m[w] > -INFINITY ? sh.warp_f[w] * fast_exp2((sh.warp_m[w] - top) * LOG2E) : sh.warp_f[w];
      mine[0] = top;
      mine[1] = total;
    }
    const int n = sh.list_n;
    if (n <= LIST) {
      // what reaches the bound of all tiles (all of it, where that is -inf), in order: each counts what is before it
      const unsigned long long* from = sh.list;
      int kept = n;
      if (tiles > 1) {
        low = bound_of(keep, beams, sh, updates & 1);
        const unsigned long long least = word_of(fmaxf(low, -FLT_MAX), 0x7fffffff);
        for (int c = tid; c < n; c += THREADS)
          if (sh.list[c] >= least) sh.kept[atomicAdd(&sh.kept_n, 1)] = sh.list[c];
        __syncthreads();
        from = sh.kept;
        kept = sh.kept_n;
      }
      for (int c = tid; c < kept; c += THREADS) {
        const unsigned long long mine_word = from[c];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < kept; ++j) place += from[j] > mine_word ? 1 : 0;
        if (place < beams) { mine[2 + 2 * place] = logit_of(mine_word); mine[3 + 2 * place] = __int_as_float(token_of(mine_word)); }
      }
      // (fewer than `beams` that may be chosen: all of them are there, the bound is -inf)
      for (int c = kept + tid; c < beams; c += THREADS) { mine[2 + 2 * c] = -INFINITY; mine[3 + 2 * c] = 0.f; }
    } else {
      // one after another: the best that comes behind the last one. (A word orders by logit, then by the lower token.)
      unsigned long long last = ~0ull;
      for (int c = 0; c < beams; ++c) {
        unsigned long long best = 0;
        for (int i = lo + tid; i < hi; i += THREADS) {
          const float value = x[i];
          if (value > -INFINITY) {
            const unsigned long long word = word_of(value, i);
            if (word < last && word > best && !is_stop(i)) best = word;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        if (tid == 0) sh.best[c & 1] = 0;
        __syncthreads();
        if (lane == 0) atomicMax(&sh.best[c & 1], best);
        __syncthreads();
        last = sh.best[c & 1];
        if (tid == 0) {
          mine[2 + 2 * c] = last ? logit_of(last) : -INFINITY;
          mine[3 + 2 * c] = __int_as_float(last ? token_of(last) : 0);
        }
      }
    }
  }
  // ---- who is last?
  __syncthreads();
  if (tid == 0) {
    // Acquire and release in one: what the block has written, which the barrier has shown to this thread, and what the others have
    // (fences before and after the ticket 8.2 us, 7.9: 1 x 4 beams of 49,152 logits).
    unsigned before;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.tickets + b) : "memory");
    sh.last = before == (unsigned)(a.beams_in * parts - 1);
    sh.list_n = sh.kept_n = 0;
  }
  __syncthreads();
  if (!sh.last) return;
  if (tid == 0) a.tickets[b] = 0u;
  // Everything that is needed is asked for at once.
  const size_t entry = 2 + 2 * (size_t)beams;
  const float* all = a.scratch + (size_t)b * a.beams_in * parts * entry;
  const int n_lists = a.beams_in * parts, n_entries = n_lists * beams;
  // (quotients by products: exact while dividend x divisor < 2^32)
  const unsigned by_beams = 0xffffffffu / (unsigned)beams + 1u, by_parts = 0xffffffffu / (unsigned)parts + 1u;
  auto list_of = [&](int c) { return beams == 1 ? c : (int)__umulhi((unsigned)c, by_beams); };
  auto beam_of = [&](int c) { return parts == 1 ? list_of(c) : (int)__umulhi((unsigned)list_of(c), by_parts); };
  auto pair_at = [&](int c) {
    const int list = list_of(c);
    return __ldcg(reinterpret_cast<const float2*>(all + (size_t)list * entry + 2 + 2 * (c - list * beams)));
  };
  constexpr int HELD = 4;  // entries stay with a thread, where they are not more than that
  const bool by_lists = n_entries > HELD * THREADS;
  const int n_held = by_lists ? 0 : n_entries;
  float2 held[HELD];
#pragma unroll
  for (int u = 0; u < HELD; ++u) held[u] = tid + u * THREADS < n_held ? pair_at(tid + u * THREADS) : make_float2(-INFINITY, 0.f);
  const bool may_end = step >= a.min_tokens;
  const int n_stop = may_end ? a.beams_in * n_stops : 0;  // (at most THREADS)
  int stop_beam = 0, stop_token = -1;
  float stop_logit = -INFINITY;
  if (tid < n_stop) {
    stop_beam = tid / n_stops;
    const int s = tid - stop_beam * n_stops;
    stop_token = sh.stops[s];
    for (int j = 0; j < s; ++j) stop_token = sh.stops[j] == stop_token ? -1 : stop_token;  // (one named twice counts once)
    if (stop_token >= 0 && stop_token < vocab) stop_logit = a.logits[(size_t)(b * a.beams_in + stop_beam) * a.row_stride + stop_token];
  }
  const bool on = warp == 0 && lane < beams;  // the first warp has a lane a beam
  const size_t at = (size_t)b * beams + lane;
  const float pool = on ? a.finished[at] : -INFINITY;
  const int pool_step = on ? a.finished_at[2 * at] : -1, pool_beam = on ? a.finished_at[2 * at + 1] : -1;
  const float length = powf((float)(step + 1), a.penalty);
  // the rows' sums: a warp a row
  for (int r = warp; r < a.beams_in; r += THREADS / 32) {
    const float score = a.scores[(size_t)b * a.beams_in + r];
    float2 part_ml = lane < parts ? __ldcg(reinterpret_cast<const float2*>(all + ((size_t)r * parts + lane) * entry)) : make_float2(-INFINITY, 0.f);
    float m = -INFINITY, sum = 0.f;
    if (score > -INFINITY) {
      m = part_ml.x;
      sum = part_ml.y;
      for (int p = lane + 32; p < parts; p += 32) {
        part_ml = __ldcg(reinterpret_cast<const float2*>(all + ((size_t)r * parts + p) * entry));
        const float m_new = fmaxf(m, part_ml.x), shift = m_new > -INFINITY ? m_new : 0.f;
        sum = (m > -INFINITY ? sum * expf(m - shift) : sum) + (part_ml.x > -INFINITY ? part_ml.y * expf(part_ml.x - shift) : part_ml.y);
        m = m_new;
      }
    }
    const float top = warp_max(m);
    sum = warp_sum(m > -INFINITY ? sum * expf(m - top) : sum);  // (0 where there is nothing, or a NaN)
    if (lane == 0) {
      sh.lse[r] = top + logf(sum);
      sh.score[r] = score > -INFINITY ? score : -INFINITY;
    }
  }
  for (int c = tid; c < beams; c += THREADS) {
    sh.chosen[c] = Candidate{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
    sh.chosen_total[c] = -INFINITY;
  }
  __syncthreads();
  // a total, -inf where the row has none (what a row without a score left in scratch is not looked at)
  auto total_of = [&](float logit, int beam) {
    const float total = (logit - sh.lse[beam]) + sh.score[beam];
    return sh.score[beam] > -INFINITY && total > -INFINITY ? total : -INFINITY;
  };
  auto candidate_at = [&](int c) {
    const float2 pair = pair_at(c);
    const int beam = beam_of(c);
    return Candidate{total_of(pair.x, beam), pair.x, beam, __float_as_int(pair.y)};
  };
  float top = -INFINITY, totals[HELD];
#pragma unroll
  for (int u = 0; u < HELD; ++u) {
    const int c = tid + u * THREADS;
    totals[u] = c < n_held ? total_of(held[u].x, beam_of(c)) : -INFINITY;
    top = fmaxf(top, totals[u]);
  }
  if (by_lists)  // (the lists' firsts alone)
    for (int list = tid; list < n_lists; list += THREADS) top = fmaxf(top, candidate_at(list * beams).total);
  if (tid < n_stop) {
    const float total = stop_token >= 0 && stop_token < vocab ? total_of(stop_logit, stop_beam) : -INFINITY;
    sh.stop[tid] = Candidate{total, stop_logit, stop_beam, stop_token};
    sh.stop_total[tid] = total;
  }
  const float low = bound_of(top, beams, sh, 0), floor_ = fmaxf(low, -FLT_MAX);
  auto offer = [&](const Candidate& one) {
    const int to = atomicAdd(&sh.list_n, 1);
    if (to < LIST) {
      sh.list[to] = ((unsigned long long)__float_as_uint(one.logit) << 32) | (unsigned)one.token;
      sh.list_total[to] = one.total;
      sh.list_beam[to] = one.beam;
    }
  };
#pragma unroll
  for (int u = 0; u < HELD; ++u)
    if (totals[u] >= floor_) offer(Candidate{totals[u], held[u].x, beam_of(tid + u * THREADS), __float_as_int(held[u].y)});
  if (by_lists) {  // (at most LIST of them: parts_for.) A list is in order: one whose first does not reach the bound has nothing that does
    for (int list = tid; list < n_lists; list += THREADS)
      if (candidate_at(list * beams).total >= floor_) sh.kept[atomicAdd(&sh.kept_n, 1)] = list;
    __syncthreads();
    const int n = sh.kept_n * beams;
    for (int c = tid; c < n; c += THREADS) {
      const int list = list_of(c);
      const Candidate one = candidate_at((int)sh.kept[list] * beams + c - list * beams);
      if (one.total >= floor_) offer(one);
    }
  }
  __syncthreads();
  auto listed = [&](int c) {
    return Candidate{sh.list_total[c], __uint_as_float((unsigned)(sh.list[c] >> 32)), sh.list_beam[c], (int)(unsigned)sh.list[c]};
  };
  const int n = sh.list_n;
  if (n <= LIST) {
    for (int c = tid; c < n; c += THREADS) {
      const float total = sh.list_total[c];
      int place = 0, equal = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        place += sh.list_total[j] > total ? 1 : 0;
        equal += sh.list_total[j] == total ? 1 : 0;
      }
      const Candidate one = listed(c);
      if (equal > 1)
        for (int j = 0; j < n; ++j) place += sh.list_total[j] == total && before(listed(j), one) ? 1 : 0;
      if (place < beams) {
        sh.chosen[place] = one;
        sh.chosen_total[place] = total;
      }
    }
  } else {
    // one after another, in the order of (total, beam, logit, token)
    Candidate last{INFINITY, INFINITY, -1, -1};
    for (int c = 0; c < beams; ++c) {
      Candidate best{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
      for (int e = tid; e < n_entries; e += THREADS) {
        const Candidate one = candidate_at(e);
        if (one.total > -INFINITY && (c == 0 || before(last, one)) && before(one, best)) best = one;
      }
      auto put = [&](const Candidate& one) {
        sh.list[tid] = ((unsigned long long)__float_as_uint(one.logit) << 32) | (unsigned)one.token;
        sh.list_total[tid] = one.total;
        sh.list_beam[tid] = one.beam;
      };
      put(best);
      __syncthreads();
      for (int o = THREADS / 2; o > 0; o >>= 1) {
        if (tid < o && before(listed(tid + o), listed(tid))) put(listed(tid + o));
        __syncthreads();
      }
      last = listed(0);
      if (tid == 0) {
        sh.chosen[c] = last;
        sh.chosen_total[c] = last.total;
      }
      __syncthreads();
    }
  }
  __syncthreads();
  // ---- texts that end: stop tokens among the first `beams` of all candidates, in order
  if (tid < n_stop) {
    const float total = sh.stop_total[tid];
    if (total > -INFINITY && total >= sh.chosen_total[beams - 1]) {
      int stops_before = 0, live_before = 0, equal = 0;
#pragma unroll 8
      for (int j = 0; j < n_stop; ++j) {
        stops_before += sh.stop_total[j] > total ? 1 : 0;
        equal += sh.stop_total[j] == total ? 1 : 0;
      }
#pragma unroll 8
      for (int j = 0; j < beams; ++j) {
        live_before += sh.chosen_total[j] > total ? 1 : 0;
        equal += sh.chosen_total[j] == total ? 1 : 0;
      }
      const Candidate one = sh.stop[tid];
      if (equal > 1) {
        for (int j = 0; j < n_stop; ++j) stops_before += sh.stop_total[j] == total && before(sh.stop[j], one) ? 1 : 0;
        for (int j = 0; j < beams; ++j) live_before += sh.chosen_total[j] == total && before(sh.chosen[j], one) ? 1 : 0;
      }
      if (stops_before + live_before < beams) {
        sh.ended[stops_before] = Candidate{total / length, one.logit, one.beam, one.token};
        atomicAdd(&sh.n_ended, 1);
      }
    }
  }
  __syncthreads();
  if (warp) return;
  // ---- places and pool: a lane a beam
  const Candidate one = on ? sh.chosen[lane] : Candidate{-INFINITY, -INFINITY, 0x7fffffff, 0};
  const bool live = on && one.total > -INFINITY;
  const unsigned same = __match_any_sync(0xffffffffu, live ? one.beam : -1 - lane);
  const bool stays = live && one.beam < beams && (same & ((1u << lane) - 1u)) == 0u;
  const unsigned taken = __reduce_or_sync(0xffffffffu, stays ? 1u << one.beam : 0u);
  const unsigned others = __ballot_sync(0xffffffffu, on && !stays);
  int place = one.beam;
  if (on && !stays) {
    unsigned free_places = ~taken;
    for (int rank = __popc(others & ((1u << lane) - 1u)); rank > 0; --rank) free_places &= free_places - 1u;
    place = __ffs(free_places) - 1;
  }
  if (on) {
    const size_t to = (size_t)b * beams + place;
    const int parent = live ? one.beam : min(place, a.beams_in - 1);
    a.scores_out[to] = live ? one.total : -INFINITY;
    a.parents[to] = parent;
    a.tokens[to] = live ? one.token : 0;
    if (history) history[place] = parent;
  }
  const int n_ended = sh.n_ended;
  int pool_place = lane, ended_place = lane;
  const float ended = lane < n_ended ? sh.ended[lane].total : -INFINITY;
  if (n_ended) {
    for (int j = 0; j < n_ended; ++j) pool_place += sh.ended[j].total > pool ? 1 : 0;
    for (int j = 0; j < beams; ++j) ended_place += __shfl_sync(0xffffffffu, pool, j) >= ended ? 1 : 0;
  }
  __syncwarp();
  float worst = -INFINITY;
  if (on && pool_place < beams) {
    const size_t to = (size_t)b * beams + pool_place;
    a.finished_out[to] = pool;
    a.finished_at_out[2 * to] = pool_step;
    a.finished_at_out[2 * to + 1] = pool_beam;
    if (pool_place == beams - 1) worst = pool;
  }
  if (lane < n_ended && ended_place < beams) {
    const size_t to = (size_t)b * beams + ended_place;
    a.finished_out[to] = ended;
    a.finished_at_out[2 * to] = step;
    a.finished_at_out[2 * to + 1] = sh.ended[lane].beam;
    if (ended_place == beams - 1) worst = ended;
  }
  worst = warp_max(worst);
  const float best = warp_max(live ? one.total : -INFINITY);
  if (lane == 0)
    a.done_out[b] = (worst > -INFINITY && (a.early || worst >= best / length)) || best == -INFINITY ? 1 : 0;
}

// Stretches a row is cut into: as many as fill the device, one more where a quarter of it would stay idle, as many more as save a
// tile where a tenth of them have to wait; of 2,048 logits at least, and not more than a warp joins at once while they are a tile
// at most. (us on 128,256 logits: 304 rows, one or two stretches, 45.7 and 34.0, 352 rows 58.1 and 52.7, 496 rows 50.1 and 53.0; 160
// rows, three or four, 26.1 and 22.4; 80 rows, seven or eight, 19.4 and 17.2; 64 rows, nine or sixteen, 17.5 and 17.4; 16 rows, 37
// or 16 to 32, 12.2 and 10.9; 4 rows, 63 or 16 to 32, 9.5 and 9.0. Of 49,152: 304 rows 26.3 and 21.2, 200 rows, two or three, 18.5 and 16.0,
// 40 rows, 14 or 15, 11.9 and 13.7.)
int parts_for(int rows, int vocab) {
  constexpr int TILE = THREADS * 4 * 8;
  int wanted = PLACES / (rows < PLACES ? rows : PLACES);
  if (4ll * wanted * rows <= 3 * PLACES) ++wanted;
  const int tiles = (vocab - 1) / (wanted * TILE) + 1;
  if (tiles > 1) {
    const int more = (vocab - 1) / ((tiles - 1) * TILE) + 1;
    if (10ll * more * rows <= 11 * PLACES) wanted = more;
  }
  const int each = (vocab - 1) / TILE + 1, most = (vocab - 1) / 2048 + 1, enough = each > 32 ? each : 32;
  if (wanted > most) wanted = most;
  return wanted < enough ? wanted : enough;
}

template <int REG>
int launch(const Args& a, int sequences, int parts, cudaStream_t stream) {
  dim3 grid(parts, sequences * a.beams_in), block(THREADS);
  return dllm_launch_pdl(select_kernel<REG>, grid, block, 0, stream, a);
}
}  // namespace

// Stretches that each of `rows` rows of `vocab` logits is cut into: scratch holds rows x stretches x (2 + 2 beams) floats.
DLLM_EXPORT int dllm_beam_select_parts(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return DLLM_BAD_ARGUMENT;
  return parts_for(rows, vocab);
}

// See the head of the file. `logits` [sequences * beams_in, vocab] with a row stride; `scores` [sequences, beams_in]; finished,
// finished_at (step, beam) and done [sequences, beams], [.., 2], [sequences], in and out (the same buffers if the caller
// likes); produced[0] + steps[0] (steps may be null): tokens the beams have; `history` (may be null): parents are also kept
// at history[steps[0]]. One structure, `bytes` long: the caller packs it at once, where every argument by itself costs a tenth
// of a microsecond (28 of them 3.4 us, packed 0.7).
struct DllmBeamSelect {
  const float* logits;
  long long row_stride;
  const float *scores, *finished;
  const int *finished_at, *done, *produced, *steps, *stop_ids;
  float *scores_out, *finished_out;
  int *finished_at_out, *done_out, *parents, *tokens, *history;
  float* scratch;
  unsigned* tickets;
  cudaStream_t stream;
  int n_stops, history_steps, sequences, beams_in, beams, vocab, min_tokens, early;
  float penalty;
};
DLLM_EXPORT int dllm_beam_select(const DllmBeamSelect* call, int bytes) {
  if (bytes != (int)(offsetof(DllmBeamSelect, penalty) + sizeof(float))) return DLLM_BAD_ARGUMENT;
  const DllmBeamSelect& c = *call;
  const int sequences = c.sequences, beams_in = c.beams_in, beams = c.beams, vocab = c.vocab, n_stops = c.n_stops;
  if (sequences <= 0) return DLLM_OK;
  if (beams_in <= 0 || beams <= 0 || vocab <= 0 || n_stops < 0 || (n_stops > 0 && !c.stop_ids) || c.row_stride < vocab || !c.produced)
    return DLLM_BAD_ARGUMENT;
  if (beams_in > MAX_BEAMS || beams > MAX_BEAMS || n_stops > MAX_STOPS || (long long)sequences * beams_in > 65535)
    return DLLM_UNSUPPORTED_SIZE;
  const int rows = sequences * beams_in, parts = parts_for(rows, vocab);
  Args a{c.logits, c.row_stride, c.scores, c.finished, c.finished_at, c.done, c.produced, c.steps, c.stop_ids, c.scores_out,
         c.finished_out, c.finished_at_out, c.done_out, c.parents, c.tokens, c.history, c.scratch, c.tickets, beams_in, beams,
         vocab, n_stops, c.min_tokens, c.early, 0, c.history_steps, c.penalty};
  a.stretch = ((vocab - 1) / parts + 4) / 4 * 4;  // stretches of one length, whole fours
  return a.stretch <= THREADS * 8 ? launch<2>(a, sequences, parts, c.stream) : launch<8>(a, sequences, parts, c.stream);
}
