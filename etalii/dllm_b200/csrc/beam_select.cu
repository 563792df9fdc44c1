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
//   1. A block takes a stretch of a row, at most 16,384 logits that stay in its threads' registers. The threads form
//      GROUPS groups, at least as many as there are beams; the smallest of the groups' maxima is a bound that at least
//      `beams` logits reach and few do: of logits in any order all groups' maxima lie within the best GROUPS H(GROUPS),
//      about 54 of 16 groups and 130 of 32. What reaches it goes to a list, and each entry counts what is before it.
//      A list that does not hold them all (many equal logits) is given up for `beams` passes over the registers.
//      The sum of exponentials goes by the block's own maximum.
//   2. The block that finishes last for its sequence (a ticket counter; nobody waits) joins the stretches' sums,
//      makes the totals and chooses among the stretches' lists the same way; a warp deals out places and pool.
// Bound by HBM where the rows are many, by the latency of the two steps where they are few.
#include "common.cuh"

namespace {
constexpr int THREADS = 512;
constexpr int MAX_BEAMS = 32, MAX_STOPS = 8;
constexpr int LIST = 1024;       // candidates a block orders by counting
constexpr int MAX_REG = 8;       // float4 a thread holds of its stretch

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
  float list_x[LIST];
  int list_t[LIST];
  float list_total[LIST];
  int list_beam[LIST];
  float group_max[THREADS / 32][MAX_BEAMS];
  float warp_f[THREADS / 32];
  int list_n, last;
  unsigned long long best[2];
  float lse[MAX_BEAMS], score[MAX_BEAMS];
  Candidate chosen[MAX_BEAMS];
  Candidate stop[MAX_BEAMS * MAX_STOPS];
  Candidate ended[MAX_BEAMS];
  int n_ended;
  int stops[MAX_STOPS];
};

__device__ __forceinline__ unsigned ordered(float v) {  // larger floats have larger words; no NaN comes here
  unsigned b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The smallest of the groups' maxima of v, and the block's largest: every thread gets both. A thread belongs to group
// threadIdx.x % GROUPS, so that a short stretch has something of every group.
template <int GROUPS>
__device__ __forceinline__ float bound_of(float v, Shared& sh, float& largest) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o >= GROUPS; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane < GROUPS) sh.group_max[threadIdx.x >> 5][lane] = v;
  __syncthreads();
  float low = -INFINITY;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) low = fmaxf(low, sh.group_max[w][lane % GROUPS]);
  largest = warp_max(low);
#pragma unroll
  for (int o = GROUPS / 2; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  return low;
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

template <int REG, int GROUPS>
__global__ void __launch_bounds__(THREADS, 2) select_kernel(const Args a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, b = row / a.beams_in, k = row % a.beams_in;
  const int part = blockIdx.x, parts = gridDim.x;
  const int beams = a.beams, vocab = a.vocab;
  if (tid == 0) { sh.list_n = 0; sh.n_ended = 0; }
  pdl_launch_dependents();
  pdl_wait();
  const int run_step = a.steps ? a.steps[0] : 0, sequences = gridDim.y / a.beams_in;
  const int step = a.produced[0] + run_step;
  // where the parents of this step are kept too
  int* history = a.history && run_step < a.history_steps ? a.history + ((size_t)run_step * sequences + b) * beams : nullptr;
  if (a.done[b]) {
    if (k == 0 && part == 0) leave_as_is(a, b, history);
    return;
  }
  if (tid < a.n_stops) {
    int id = a.stop_ids[tid];
    for (int s = 0; s < tid; ++s) id = a.stop_ids[s] == id ? -1 : id;  // (one named twice counts once)
    sh.stops[tid] = id;
  }
  float* mine = a.scratch + ((size_t)row * parts + part) * (2 + 2 * beams);
  if (a.scores[(size_t)b * a.beams_in + k] > -INFINITY) {
    // ---- the stretch, in registers
    const float* x = a.logits + (size_t)row * a.row_stride;
    const int lo = part * a.stretch, hi = min(vocab, lo + a.stretch);
    // pieces of four begin where addresses are multiples of 16 bytes
    const int skew = (int)((reinterpret_cast<uintptr_t>(x + lo) >> 2) & 3);
    float v[4 * REG];
#pragma unroll
    for (int r = 0; r < REG; ++r) {
      int i = lo - skew + 4 * (r * THREADS + tid);
      if (i >= lo && i + 3 < hi) {
        float4 four = __ldcs(reinterpret_cast<const float4*>(x + i));
        v[4 * r] = four.x; v[4 * r + 1] = four.y; v[4 * r + 2] = four.z; v[4 * r + 3] = four.w;
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u) v[4 * r + u] = i + u >= lo && i + u < hi ? __ldcs(x + i + u) : -INFINITY;
      }
    }
    __syncthreads();  // (the stop tokens are there)
    const int n_stops = a.n_stops;
    float top = -INFINITY, keep = -INFINITY;  // of all logits; of those that may be chosen
#pragma unroll
    for (int r = 0; r < REG; ++r) {
      float four = fmaxf(fmaxf(v[4 * r], v[4 * r + 1]), fmaxf(v[4 * r + 2], v[4 * r + 3]));
      top = fmaxf(top, four);
    }
    keep = top;
    if (n_stops) {  // a thread whose piece holds a stop token looks closer
      bool holds = false;
      for (int s = 0; s < n_stops; ++s) {
        int at = sh.stops[s] - (lo - skew);
        holds = holds || (sh.stops[s] >= lo && sh.stops[s] < hi && (at >> 2) % THREADS == tid);
      }
      if (holds) {
        keep = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4 * REG; ++e) {
          int i = lo - skew + 4 * ((e >> 2) * THREADS + tid) + (e & 3);
          bool stop = false;
          for (int s = 0; s < n_stops; ++s) stop = stop || sh.stops[s] == i;
          if (!stop) keep = fmaxf(keep, v[e]);
        }
      }
    }
    float unused, m;
    {  // the block's maximum over everything, for the sum
      float t = warp_max(top);
      if (lane == 0) sh.warp_f[warp] = t;
    }
    const float low = bound_of<GROUPS>(keep, sh, unused);
    m = sh.warp_f[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, sh.warp_f[w]);
    auto is_stop = [&](int i) {
      bool stop = false;
      for (int s = 0; s < n_stops; ++s) stop = stop || sh.stops[s] == i;
      return stop;
    };
    float sum = 0.f;
    const float shift = m > -INFINITY ? m : 0.f;  // (a stretch of nothing but -inf adds nothing)
#pragma unroll
    for (int e = 0; e < 4 * REG; ++e) {
      sum += expf(v[e] - shift);
      if (v[e] >= low && v[e] > -INFINITY) {
        int i = lo - skew + 4 * ((e >> 2) * THREADS + tid) + (e & 3);
        if (!is_stop(i)) {
          int at = atomicAdd(&sh.list_n, 1);
          if (at < LIST) { sh.list_x[at] = v[e]; sh.list_t[at] = i; }
        }
      }
    }
    sum = warp_sum(sum);
    __syncthreads();  // (everybody has read the maxima; the list is whole)
    if (lane == 0) sh.warp_f[warp] = sum;
    const int n = sh.list_n;
    if (n <= LIST) {
      for (int c = tid; c < n; c += THREADS) {
        float xc = sh.list_x[c];
        int tc = sh.list_t[c], place = 0;
        for (int j = 0; j < n; ++j) {
          float xj = sh.list_x[j];
          place += xj > xc ? 1 : 0;
          if (xj == xc && j != c) place += sh.list_t[j] < tc ? 1 : 0;
        }
        if (place < beams) { mine[2 + 2 * place] = xc; mine[3 + 2 * place] = __int_as_float(tc); }
      }
      for (int c = n + tid; c < beams; c += THREADS) { mine[2 + 2 * c] = -INFINITY; mine[3 + 2 * c] = 0.f; }
    } else {
      // one after another: the best that comes behind the last one. (A word orders by logit, then by the lower token.)
      unsigned long long last = ~0ull;
      for (int c = 0; c < beams; ++c) {
        unsigned long long best = 0;
#pragma unroll
        for (int e = 0; e < 4 * REG; ++e) {
          int i = lo - skew + 4 * ((e >> 2) * THREADS + tid) + (e & 3);
          if (v[e] > -INFINITY) {
            unsigned long long word = ((unsigned long long)ordered(v[e]) << 32) | (unsigned)(0x7fffffff - i);
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
          unsigned w = (unsigned)(last >> 32);
          mine[2 + 2 * c] = last ? __uint_as_float(w & 0x80000000u ? w & 0x7fffffffu : ~w) : -INFINITY;
          mine[3 + 2 * c] = __int_as_float(last ? 0x7fffffff - (int)(unsigned)last : 0);
        }
      }
    }
    __syncthreads();
    if (tid == 0) {
      float total = 0.f;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) total += sh.warp_f[w];
      mine[0] = m;
      mine[1] = total;
    }
  }
  // ---- who is last?
  __threadfence();
  __syncthreads();
  if (tid == 0) sh.last = atomicAdd(&a.tickets[b], 1u) == (unsigned)(a.beams_in * parts - 1);
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  if (tid == 0) { a.tickets[b] = 0u; sh.list_n = 0; }
  const size_t entry = 2 + 2 * (size_t)beams;
  const float* all = a.scratch + (size_t)b * a.beams_in * parts * entry;
  // the rows' sums: a warp a row
  for (int r = warp; r < a.beams_in; r += THREADS / 32) {
    float score = a.scores[(size_t)b * a.beams_in + r], top = -INFINITY, sum = 0.f;
    if (score > -INFINITY) {
      for (int p = lane; p < parts; p += 32) top = fmaxf(top, __ldcg(all + ((size_t)r * parts + p) * entry));
      top = warp_max(top);
      for (int p = lane; p < parts; p += 32) {
        float pm = __ldcg(all + ((size_t)r * parts + p) * entry), ps = __ldcg(all + ((size_t)r * parts + p) * entry + 1);
        sum += pm > -INFINITY ? ps * expf(pm - top) : ps;  // (ps is 0 there, or a NaN)
      }
      sum = warp_sum(sum);
    }
    if (lane == 0) {
      sh.lse[r] = top + logf(sum);
      sh.score[r] = score > -INFINITY ? score : -INFINITY;
    }
  }
  __syncthreads();
  const int n_entries = a.beams_in * parts * beams, per_row = parts * beams;
  auto load = [&](int c) {
    Candidate out;
    out.beam = c / per_row;
    out.total = -INFINITY;
    out.logit = -INFINITY;
    out.token = 0;
    if (sh.score[out.beam] > -INFINITY) {
      const float* at = all + (size_t)(c / beams) * entry + 2 + 2 * (c % beams);
      float2 pair = __ldcg(reinterpret_cast<const float2*>(at));
      out.logit = pair.x;
      out.token = __float_as_int(pair.y);
      float total = (pair.x - sh.lse[out.beam]) + sh.score[out.beam];
      if (total > -INFINITY) out.total = total;
    }
    return out;
  };
  float top = -INFINITY, unused;
  for (int c = tid; c < n_entries; c += THREADS) top = fmaxf(top, load(c).total);
  const float low = bound_of<GROUPS>(top, sh, unused);
  for (int c = tid; c < n_entries; c += THREADS) {
    Candidate one = load(c);
    if (one.total >= low && one.total > -INFINITY) {
      int at = atomicAdd(&sh.list_n, 1);
      if (at < LIST) {
        sh.list_x[at] = one.logit;
        sh.list_t[at] = one.token;
        sh.list_total[at] = one.total;
        sh.list_beam[at] = one.beam;
      }
    }
  }
  // the totals of the stop tokens, where they may end a text
  const bool may_end = step >= a.min_tokens;
  const int n_stop = may_end ? a.beams_in * a.n_stops : 0;
  for (int c = tid; c < n_stop; c += THREADS) {
    Candidate one{-INFINITY, -INFINITY, c / a.n_stops, sh.stops[c % a.n_stops]};
    if (sh.score[one.beam] > -INFINITY && one.token >= 0 && one.token < vocab) {
      one.logit = a.logits[(size_t)(b * a.beams_in + one.beam) * a.row_stride + one.token];
      float total = (one.logit - sh.lse[one.beam]) + sh.score[one.beam];
      if (total > -INFINITY) one.total = total;
    }
    sh.stop[c] = one;
  }
  for (int c = tid; c < beams; c += THREADS) sh.chosen[c] = Candidate{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
  __syncthreads();
  const int n = sh.list_n;
  if (n <= LIST) {
    for (int c = tid; c < n; c += THREADS) {
      Candidate one{sh.list_total[c], sh.list_x[c], sh.list_beam[c], sh.list_t[c]};
      int place = 0;
      for (int j = 0; j < n; ++j) {
        float total = sh.list_total[j];
        place += total > one.total ? 1 : 0;
        if (total == one.total && j != c) place += before(Candidate{total, sh.list_x[j], sh.list_beam[j], sh.list_t[j]}, one) ? 1 : 0;
      }
      if (place < beams) sh.chosen[place] = one;
    }
  } else {
    // one after another, in the order of (total, beam, logit, token): a round finds the best total behind the last one, and
    // what shares it goes by a second word
    Candidate last{INFINITY, INFINITY, -1, -1};
    for (int c = 0; c < beams; ++c) {
      Candidate best{-INFINITY, -INFINITY, 0x7fffffff, 0x7fffffff};
      for (int e = tid; e < n_entries; e += THREADS) {
        Candidate one = load(e);
        if (one.total > -INFINITY && (c == 0 || before(last, one)) && before(one, best)) best = one;
      }
      sh.list_total[tid] = best.total;
      sh.list_x[tid] = best.logit;
      sh.list_beam[tid] = best.beam;
      sh.list_t[tid] = best.token;
      __syncthreads();
      for (int o = THREADS / 2; o > 0; o >>= 1) {
        if (tid < o) {
          Candidate one{sh.list_total[tid], sh.list_x[tid], sh.list_beam[tid], sh.list_t[tid]};
          Candidate other{sh.list_total[tid + o], sh.list_x[tid + o], sh.list_beam[tid + o], sh.list_t[tid + o]};
          if (before(other, one)) {
            sh.list_total[tid] = other.total;
            sh.list_x[tid] = other.logit;
            sh.list_beam[tid] = other.beam;
            sh.list_t[tid] = other.token;
          }
        }
        __syncthreads();
      }
      last = Candidate{sh.list_total[0], sh.list_x[0], sh.list_beam[0], sh.list_t[0]};
      if (tid == 0) sh.chosen[c] = last;
      __syncthreads();
    }
  }
  __syncthreads();
  // ---- texts that end: stop tokens among the first `beams` of all candidates, in order
  const float length = powf((float)(step + 1), a.penalty);
  for (int c = tid; c < n_stop; c += THREADS) {
    Candidate one = sh.stop[c];
    if (!(one.total > -INFINITY)) continue;
    int stops_before = 0, live_before = 0;
    for (int j = 0; j < n_stop; ++j) stops_before += before(sh.stop[j], one) ? 1 : 0;
    for (int j = 0; j < beams; ++j) live_before += sh.chosen[j].total > -INFINITY && before(sh.chosen[j], one) ? 1 : 0;
    if (stops_before + live_before < beams) {
      sh.ended[stops_before] = Candidate{one.total / length, one.logit, one.beam, one.token};
      atomicAdd(&sh.n_ended, 1);
    }
  }
  __syncthreads();
  if (warp) return;
  // ---- places and pool: a lane a beam
  const size_t at = (size_t)b * beams + lane;
  const bool on = lane < beams;
  Candidate one = on ? sh.chosen[lane] : Candidate{-INFINITY, -INFINITY, 0x7fffffff, 0};
  const bool live = on && one.total > -INFINITY;
  unsigned same = __match_any_sync(0xffffffffu, live ? one.beam : -1 - lane);
  const bool stays = live && one.beam < beams && (same & ((1u << lane) - 1u)) == 0u;
  unsigned taken = __reduce_or_sync(0xffffffffu, stays ? 1u << one.beam : 0u);
  unsigned others = __ballot_sync(0xffffffffu, on && !stays);
  int place = one.beam;
  if (on && !stays) {
    int rank = __popc(others & ((1u << lane) - 1u));
    place = 0;
    for (int i = 0; i < beams; ++i) {
      if (taken >> i & 1u) continue;
      if (rank-- == 0) { place = i; break; }
    }
  }
  if (on) {
    size_t to = (size_t)b * beams + place;
    int parent = live ? one.beam : min(place, a.beams_in - 1);
    a.scores_out[to] = live ? one.total : -INFINITY;
    a.parents[to] = parent;
    a.tokens[to] = live ? one.token : 0;
    if (history) history[place] = parent;
  }
  const int n_ended = sh.n_ended;
  float pool = on ? a.finished[at] : -INFINITY;
  int pool_step = on ? a.finished_at[2 * at] : -1, pool_beam = on ? a.finished_at[2 * at + 1] : -1;
  int pool_place = lane, ended_place = lane;
  float ended = lane < n_ended ? sh.ended[lane].total : -INFINITY;
  for (int j = 0; j < n_ended; ++j) pool_place += sh.ended[j].total > pool ? 1 : 0;
  for (int j = 0; j < beams; ++j) ended_place += __shfl_sync(0xffffffffu, pool, j) >= ended ? 1 : 0;
  __syncwarp();
  float worst = -INFINITY;
  if (on && pool_place < beams) {
    size_t to = (size_t)b * beams + pool_place;
    a.finished_out[to] = pool;
    a.finished_at_out[2 * to] = pool_step;
    a.finished_at_out[2 * to + 1] = pool_beam;
    if (pool_place == beams - 1) worst = pool;
  }
  if (lane < n_ended && ended_place < beams) {
    size_t to = (size_t)b * beams + ended_place;
    a.finished_out[to] = ended;
    a.finished_at_out[2 * to] = step;
    a.finished_at_out[2 * to + 1] = sh.ended[lane].beam;
    if (ended_place == beams - 1) worst = ended;
  }
  worst = warp_max(worst);
  float best = warp_max(live ? one.total : -INFINITY);
  if (lane == 0)
    a.done_out[b] = (worst > -INFINITY && (a.early || worst >= best / length)) || best == -INFINITY ? 1 : 0;
}

// Logits a thread holds (in fours): enough blocks to fill the device where the rows are few, long stretches where they are
// many.
int registers_for(int rows, int vocab) {
  for (int reg = MAX_REG; reg > 1; reg >>= 1)
    if ((long long)rows * ((vocab + THREADS * 4 * reg - 1) / (THREADS * 4 * reg)) >= 2 * 148) return reg;
  return 1;
}
// (four logits fewer than fit: a stretch may begin inside a piece of four)
int parts_for(int vocab, int reg) { return (vocab - 1) / (THREADS * 4 * reg - 4) + 1; }

template <int REG>
int launch(const Args& a, int sequences, int parts, cudaStream_t stream) {
  dim3 grid(parts, sequences * a.beams_in), block(THREADS);
  return a.beams <= 16 ? dllm_launch_pdl(select_kernel<REG, 16>, grid, block, 0, stream, a)
                       : dllm_launch_pdl(select_kernel<REG, 32>, grid, block, 0, stream, a);
}
}  // namespace

// Stretches that each of `rows` rows of `vocab` logits is cut into: scratch holds rows x stretches x (2 + 2 beams) floats.
DLLM_EXPORT int dllm_beam_select_parts(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0) return DLLM_BAD_ARGUMENT;
  return parts_for(vocab, registers_for(rows, vocab));
}

// See the head of the file. `logits` [sequences * beams_in, vocab] with a row stride; `scores` [sequences, beams_in]; finished,
// finished_at (step, beam) and done [sequences, beams], [.., 2], [sequences], in and out (the same buffers if the caller
// likes); produced[0] + steps[0] (steps may be null): tokens the beams have; `history` (may be null): parents are also kept
// at history[steps[0]].
DLLM_EXPORT int dllm_beam_select(const float* logits, long long row_stride, const float* scores, const float* finished,
                                 const int* finished_at, const int* done, const int* produced, const int* steps,
                                 const int* stop_ids, int n_stops, float* scores_out, float* finished_out,
                                 int* finished_at_out, int* done_out, int* parents, int* tokens, int* history,
                                 int history_steps, float* scratch, unsigned* tickets, int sequences, int beams_in, int beams,
                                 int vocab, int min_tokens, float penalty, int early, cudaStream_t stream) {
  if (sequences <= 0) return DLLM_OK;
  if (beams_in <= 0 || beams <= 0 || vocab <= 0 || n_stops < 0 || (n_stops > 0 && !stop_ids) || row_stride < vocab)
    return DLLM_BAD_ARGUMENT;
  if (beams_in > MAX_BEAMS || beams > MAX_BEAMS || n_stops > MAX_STOPS || (long long)sequences * beams_in > 65535)
    return DLLM_UNSUPPORTED_SIZE;
  const int rows = sequences * beams_in, reg = registers_for(rows, vocab), parts = parts_for(vocab, reg);
  Args a{logits, row_stride, scores, finished, finished_at, done, produced, steps, stop_ids, scores_out, finished_out,
         finished_at_out, done_out, parents, tokens, history, scratch, tickets, beams_in, beams, vocab, n_stops, min_tokens,
         early, 0, history_steps, penalty};
  a.stretch = ((vocab - 1) / parts + 4) / 4 * 4;  // stretches of one length, whole fours: at most THREADS * 4 * reg - 4
  switch (reg) {
    case 1: return launch<1>(a, sequences, parts, stream);
    case 2: return launch<2>(a, sequences, parts, stream);
    case 4: return launch<4>(a, sequences, parts, stream);
    default: return launch<8>(a, sequences, parts, stream);
  }
}
