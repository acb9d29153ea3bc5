// Rows of the paged caches from one place to another, every operand of every layer in one launch:
//   pg_copy_pages   the first rows of pages into other pages (a request that forks shares its full pages and owns a copy of the last one)
//   pg_keep_rows    row ctx + i <- row ctx + path[i], i < kept: the accepted path of a drafted tree moves together behind the stored rows
//
// What bounds them: bytes moved (2 rows x row bytes x operands) where many pages are copied (256 pages of 64 rows, 24 operands of 1 KB rows: 43 us, 203 MB written, the shared sources
// mostly read from L2); a launch and a few trips to memory for a single request (4 us) and for paths (48 over 16 operands of 4 KB rows 10 us).
// An operand is described once (PgPageOperand, a table on the device that a cache keeps); pieces of 16 KB go to CTAs of their own, every thread has four
// 16-byte loads under way; of a path's rows sixteen, four rows by four pieces (48 paths 10.3 us, four rows by one piece 13.8).
#include "common.cuh"
#include "paligemma_b200.h"

namespace {

constexpr int kThreads = 256, kLoads = 4, kPiece = kThreads * kLoads * 16, kMoves = 256, kCols = 64, kRowLanes = kThreads / kCols, kParts = 4;

struct Moves {
  int n;
  int at[kMoves][3];  // source page, destination page, rows
};
static_assert(sizeof(Moves) < 4000, "the moves travel as a kernel's argument");

template <typename U>
__device__ __forceinline__ void copy_run(const char* src, char* dst, long long lo, long long hi) {
  const U* s = reinterpret_cast<const U*>(src);
  U* d = reinterpret_cast<U*>(dst);
  const long long end = hi / static_cast<long long>(sizeof(U));
  for (long long i = lo / static_cast<long long>(sizeof(U)) + threadIdx.x; i < end; i += kThreads * kLoads) {
    U v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (i + k * kThreads < end) v[k] = s[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (i + k * kThreads < end) d[i + k * kThreads] = v[k];
  }
}

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const PgPageOperand* __restrict__ ops, const __grid_constant__ Moves mv, int page, int pieces) {
  pg::griddep_begin();
  const int m = blockIdx.x / pieces;
  const long long lo = static_cast<long long>(blockIdx.x % pieces) * kPiece;
  const PgPageOperand op = ops[blockIdx.y];
  const int src = mv.at[m][0], dst = mv.at[m][1], rows = min(mv.at[m][2], page);
  if (src < 0 || dst < 0 || src >= op.pages || dst >= op.pages) return;
  const char* s = static_cast<const char*>(op.base) + src * op.page_bytes;
  char* d = static_cast<char*>(op.base) + dst * op.page_bytes;
  if (op.heads > 0) {  // a byte per row and head, a head's rows side by side
    const long long hi = min(static_cast<long long>(op.heads) * rows, lo + kPiece);
    for (long long i = lo + threadIdx.x; i < hi; i += kThreads) {
      const long long at = i / rows * page + i % rows;
      d[at] = s[at];
    }
    return;
  }
  const long long hi = min(static_cast<long long>(rows) * op.row_bytes, lo + kPiece);
  if (lo >= hi) return;
  switch (op.unit) {
    case 16: copy_run<uint4>(s, d, lo, hi); break;
    case 4: copy_run<uint32_t>(s, d, lo, hi); break;
    case 2: copy_run<uint16_t>(s, d, lo, hi); break;
    default: copy_run<uint8_t>(s, d, lo, hi);
  }
}

// The columns [c0, c0 + kParts kCols) of the path's rows: kRowLanes x kLoads rows are read, then written.  Paths ascend with path[i] >= i, so what a batch writes lies in
// front of every row that is still to be read.
template <typename U>
__device__ __forceinline__ void keep_columns(const PgPageOperand& op, const int* __restrict__ table, int max_pages, const int* __restrict__ path, int kept, int ctx, int n, int page,
                                             int c0) {
  const int c = c0 + threadIdx.x % kCols, lane = threadIdx.x / kCols;
  const int cols = op.heads > 0 ? op.heads : op.row_bytes / static_cast<int>(sizeof(U));
  const long long step = kCols * (op.heads > 0 ? static_cast<long long>(page) : static_cast<long long>(sizeof(U)));  // bytes between a thread's columns
  auto place = [&](int row) -> char* {
    const int slot = row / page;
    const int id = slot < max_pages ? table[slot] : -1;
    if (id < 0 || id >= op.pages) return nullptr;
    char* p = static_cast<char*>(op.base) + id * op.page_bytes;
    return op.heads > 0 ? p + static_cast<long long>(c) * page + row % page : p + static_cast<long long>(row % page) * op.row_bytes + c * static_cast<long long>(sizeof(U));
  };
  for (int i0 = 0; i0 < kept; i0 += kRowLanes * kLoads) {
    U v[kLoads][kParts];
    char* to[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
      const int i = i0 + k * kRowLanes + lane;
      to[k] = nullptr;
      if (i < kept) {
        const int p = path[i];
        if (p > i && p < n) {  // (rows that stay where they are need no move)
          const char* from = place(ctx + p);
          to[k] = from != nullptr ? place(ctx + i) : nullptr;
          if (to[k] != nullptr)
#pragma unroll
            for (int j = 0; j < kParts; ++j)
              if (c + j * kCols < cols) v[k][j] = *reinterpret_cast<const U*>(from + j * step);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (to[k] != nullptr)
#pragma unroll
        for (int j = 0; j < kParts; ++j)
          if (c + j * kCols < cols) *reinterpret_cast<U*>(to[k] + j * step) = v[k][j];
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads) keep_rows_kernel(const PgKeepRows a, int pieces) {
  pg::griddep_begin();
  const int e = blockIdx.x / pieces, c0 = blockIdx.x % pieces * (kCols * kParts), page = a.page, max_pages = a.max_pages;
  const PgPageOperand op = a.operands[blockIdx.y];
  if (c0 >= (op.heads > 0 ? op.heads : op.row_bytes / op.unit)) return;
  const int n = a.n[e], ctx = a.ctx[e], count = min(min(a.kept[e], a.path_ld), n);
  if (count <= 0 || ctx < 0) return;
  const int* p = a.path + static_cast<long long>(e) * a.path_ld;
  const int* table = a.page_table + static_cast<long long>(e) * max_pages;
  switch (op.heads > 0 ? 1 : op.unit) {
    case 16: keep_columns<uint4>(op, table, max_pages, p, count, ctx, n, page, c0); break;
    case 4: keep_columns<uint32_t>(op, table, max_pages, p, count, ctx, n, page, c0); break;
    case 2: keep_columns<uint16_t>(op, table, max_pages, p, count, ctx, n, page, c0); break;
    default: keep_columns<uint8_t>(op, table, max_pages, p, count, ctx, n, page, c0);
  }
}

}  // namespace

extern "C" int pg_copy_pages(const PgPageOperand* operands, int count, int page, long long most_page_bytes, const int* moves_host, int moves, void* stream) {
  if (operands == nullptr || count <= 0 || count > 65535 || page <= 0 || most_page_bytes <= 0 || moves < 0 || (moves > 0 && moves_host == nullptr)) return PG_ERR_ARG;
  const long long pieces = (most_page_bytes + kPiece - 1) / kPiece;
  if (pieces * kMoves > 0x7fffffff) return PG_ERR_ARG;
  for (int at = 0; at < moves; at += kMoves) {
    Moves mv;
    mv.n = moves - at < kMoves ? moves - at : kMoves;
    for (int i = 0; i < mv.n; ++i)
      for (int k = 0; k < 3; ++k) mv.at[i][k] = moves_host[(at + i) * 3LL + k];
    if (pg::launch_kernel(copy_pages_kernel, dim3(static_cast<unsigned>(mv.n * pieces), count), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), operands, mv, page,
                          static_cast<int>(pieces)) != cudaSuccess)
      return PG_ERR_CUDA;
  }
  return PG_OK;
}

extern "C" int pg_keep_rows(const PgKeepRows* args, void* stream) {
  if (args == nullptr) return PG_ERR_ARG;
  const PgKeepRows& a = *args;
  if (a.operands == nullptr || a.count <= 0 || a.count > 65535 || a.page <= 0 || a.most_columns <= 0 || a.page_table == nullptr || a.max_pages <= 0 || a.n == nullptr ||
      a.ctx == nullptr || a.path == nullptr || a.path_ld <= 0 || a.kept == nullptr || a.entries <= 0)
    return PG_ERR_ARG;
  const long long pieces = (a.most_columns + kCols * kParts - 1) / (kCols * kParts);
  if (pieces * a.entries > 0x7fffffff) return PG_ERR_ARG;
  return pg::launch_kernel(keep_rows_kernel, dim3(static_cast<unsigned>(a.entries * pieces), a.count), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a,
                           static_cast<int>(pieces)) == cudaSuccess
             ? PG_OK
             : PG_ERR_CUDA;
}
