// Between two steps of a beam search every beam takes over what the beam that it continues keeps: the page table, the rows of
// the page that is being filled, the fixed-size states.
//
// Beams own the pages that they write, from the page that holds the end of the prompt on; a page is written while it is the
// newest and never again. With `length` positions cached, the pages below length / page_size are full: a beam takes them
// over by their numbers. Of the page at length / page_size, which is its own, it takes over the rows that are filled; the
// page's own number stays. States are copied whole. All beams of a sequence move at once, in place: a thread holds the
// same 16 (or 4) bytes of all beams that move before it writes any of them, so any permutation and any fan-out is right and
// no second buffer is needed. Beams that keep to themselves are neither read for their own sake nor written.
// Attention kernels read page tables and cached rows ahead of their wait: the kernel behind this one starts when this one is over.
//
// The work is cut into pieces that a list on the device names, made once for a cache: 32 rows of a plane (one layer's keys or
// values of one head) of the newest page, 8 KB of a state, a page table. A block moves one piece of one sequence's beams.
// Bound by HBM: what is continued is read once, what moves is written once. Measured with 8, 16, 32 and 64 rows a piece, us: 8 x 8 beams of
// 32 layers of 8 heads of 128, five of eight move, 44 rows 78.4, 65.3, 61.9, 62.0 (5.9 TB/s); 3 x 5 float32 beams in a ring, 30 layers
// of 3 heads of 64, 61 rows 20.9, 19.7, 20.2, 21.9 (1,083 blocks of 32 rows where 740 are resident: five of a multiprocessor, by registers;
// 21.0 since the next move no longer starts under this one); with 8, 16 and 32 KB of a state a piece, 4 x 4 beams with 12 states of 1 MB 34.1,
// 34.9, 36.2 (6.0 TB/s).
#include "common.cuh"

namespace {
constexpr int THREADS = 256, MAX_BEAMS = 32;

enum { ROWS = 0, STATE = 1, TABLE = 2 };

// One piece, 64 bytes (the host writes them: cache/beams.py).
struct Piece {
  char* base;             // of page 0 / slot 0 / table row 0
  long long stride;       // from one page or slot to the next, bytes
  const int* table;       // ROWS: the page table
  long long units;        // pages or slots there are
  int table_width;        // ROWS, TABLE: entries of a row
  int kind;
  int bytes;              // ROWS: of a row; STATE: of the piece
  int vector;             // bytes moved at a time: 16 or 4
  int first, count;       // ROWS: the rows of the page that the piece has
  long long unused;
};
static_assert(sizeof(Piece) == 64, "the host lays pieces out as 64 bytes");

template <typename V, int BEAMS>
__device__ __forceinline__ void move(const long long* from, char* const* to, int beams, int bytes) {
  for (int at = threadIdx.x * (int)sizeof(V); at < bytes; at += THREADS * (int)sizeof(V)) {
    V held[BEAMS];
#pragma unroll
    for (int i = 0; i < BEAMS; ++i)
      if (i < beams && from[i]) held[i] = *reinterpret_cast<const V*>(reinterpret_cast<const char*>(from[i]) + at);
#pragma unroll
    for (int i = 0; i < BEAMS; ++i)
      if (i < beams && from[i]) *reinterpret_cast<V*>(to[i] + at) = held[i];
  }
}

template <int BEAMS>
__global__ void __launch_bounds__(THREADS) reorder_kernel(const Piece* __restrict__ pieces, const int* __restrict__ slots,
                                                          const int* __restrict__ parents, const int* __restrict__ lengths,
                                                          int length_stride, int ahead, int beams, int page_size) {
  __shared__ long long from[BEAMS];  // where a beam that moves comes from, 0 for one that stays
  __shared__ char* to[BEAMS];
  const int b = blockIdx.y;
  const Piece piece = pieces[blockIdx.x];
  pdl_wait();
  const int length = lengths[(size_t)b * length_stride] + ahead;
  const int full = length / page_size;
  int bytes = piece.bytes;
  if (piece.kind == ROWS) bytes *= min(max(length % page_size - piece.first, 0), piece.count);
  if (piece.kind == TABLE) bytes = 4 * min(full, piece.table_width);
  if (bytes == 0) return;
  bool moves = false;
  if ((int)threadIdx.x < beams) {
    const int i = threadIdx.x;
    int parent = parents[b * beams + i];
    long long source = 0;
    char* target = nullptr;
    if (parent != i && parent >= 0 && parent < beams && length > 0) {
      long long here = slots[b * beams + i], there = slots[b * beams + parent];
      bool known = here >= 0 && there >= 0;
      if (piece.kind == ROWS) {
        known = known && full < piece.table_width;
        here = known ? piece.table[here * piece.table_width + full] : -1;
        there = known ? piece.table[there * piece.table_width + full] : -1;
      }
      if (here >= 0 && there >= 0 && here < piece.units && there < piece.units && here != there) {
        source = (long long)piece.base + there * piece.stride;
        target = piece.base + here * piece.stride;
      }
    }
    from[i] = source;
    to[i] = target;
    moves = source != 0;
  }
  if (!__syncthreads_or(moves)) return;
  if (piece.vector == 16) move<uint4, BEAMS>(from, to, beams, bytes);
  else move<unsigned, BEAMS>(from, to, beams, bytes);
}
}  // namespace

// See the head of the file. `pieces`: the list (device); slots, parents [sequences, beams]; a sequence's length is
// lengths[sequence * length_stride] + ahead. One structure, `bytes` long, which the caller packs at once.
struct DllmBeamReorder {
  const void* pieces;
  const int *slots, *parents, *lengths;
  cudaStream_t stream;
  int n_pieces, length_stride, ahead, sequences, beams, page_size;
};
DLLM_EXPORT int dllm_beam_reorder(const DllmBeamReorder* call, int bytes) {
  if (bytes != (int)sizeof(DllmBeamReorder)) return DLLM_BAD_ARGUMENT;
  const auto [pieces, slots, parents, lengths, stream, n_pieces, length_stride, ahead, sequences, beams, page_size] = *call;
  if (sequences <= 0 || n_pieces <= 0 || beams == 1) return DLLM_OK;
  if (beams <= 0 || page_size <= 0 || length_stride <= 0) return DLLM_BAD_ARGUMENT;
  if (beams > MAX_BEAMS || sequences > 65535) return DLLM_UNSUPPORTED_SIZE;
  dim3 grid(n_pieces, sequences), block(THREADS);
  const Piece* list = static_cast<const Piece*>(pieces);
  if (beams <= 4)
    return dllm_launch_pdl(reorder_kernel<4>, grid, block, 0, stream, list, slots, parents, lengths, length_stride, ahead, beams, page_size);
  if (beams <= 8)
    return dllm_launch_pdl(reorder_kernel<8>, grid, block, 0, stream, list, slots, parents, lengths, length_stride, ahead, beams, page_size);
  if (beams <= 16)
    return dllm_launch_pdl(reorder_kernel<16>, grid, block, 0, stream, list, slots, parents, lengths, length_stride, ahead, beams, page_size);
  return dllm_launch_pdl(reorder_kernel<32>, grid, block, 0, stream, list, slots, parents, lengths, length_stride, ahead, beams, page_size);
}
