// A paged key/value cache: what the kernels that write and read it share.
#pragma once
#include "common.cuh"

namespace bones {

// The new tokens of B sequences lie one after another in N rows: sequence b's are starts[b] .. starts[b + 1], the first at position pos[b].
// Position p of sequence b is slot p % P of page table[b * ldt + p / P]; k, v: [pages, H, P, D].
struct Paged {
  const int* starts;   // [B + 1], ascending
  const int* pos;      // [B]
  const int* table;    // [B, M], rows ldt apart
  long long ldt;
  int B, N, M, H;
  int shift;           // log2 P
  int pages;
  int cap;             // positions with a place in the table: M * P
  const void* values;  // the cache's v
};

struct Piece {
  int row, len, pos;   // its rows, and the position of the first
  int live;            // rows whose position is inside the table: the others are left out
};

__device__ __forceinline__ Piece paged_piece(const Paged& p, int b) {
  Piece s;
  s.row = min(max(p.starts[b], 0), p.N);
  s.len = min(max(p.starts[b + 1], s.row), p.N) - s.row;
  s.pos = p.pos[b];
  s.live = s.pos < 0 || s.pos >= p.cap ? 0 : min(s.len, p.cap - s.pos);
  return s;
}

// The sequence that row r belongs to, by a warp: the number of starts at or before r, less one (-1 in front of the first, B behind the last).
template <typename I, typename R>
__device__ __forceinline__ int paged_owner(const I* starts, int B, R r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = B + 1;                         // how many starts are <= r lies in [lo, hi]
  while (hi - lo > 32) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step - 1;     // the last one of the lane's share
    const int full = __popc(__ballot_sync(0xffffffffu, i < hi && starts[min(i, B)] <= r));
    const int from = lo + full * step;
    hi = min(hi, from + step);
    lo = min(from, hi);
  }
  const int i = lo + lane;
  return lo + __popc(__ballot_sync(0xffffffffu, i < hi && starts[min(i, B)] <= r)) - 1;
}

// First row's offset of page `id`, head h; -1 where there is no such page.
__device__ __forceinline__ long long paged_at(const Paged& p, int id, int h) {
  return id < 0 || id >= p.pages ? -1 : ((long long)id * p.H + h) << p.shift;
}

constexpr int MOST_WINDOW = 1 << 24;   // tiles of 128 tokens that hide none of any cache's

// Host: attention of longer pieces (paged_pieces.cu) and the bytes that it works with.
int paged_pieces(const void* q, const void* k, const Paged& p, const int* doc_start, void* y, int D, float scale, int window_tiles, int sms, void* work, void* stream);
long long paged_pieces_room(int B, int N, int cap, int H, int D, int window_tiles, int sms);

// Host: whether a call is not one that the kernels are made for.
inline bool paged_refused(int B, int N, int M, int H, int D, int shift, int pages, long long ldt, const void* k, const void* v, const int* starts, const int* pos,
                          const int* table) {
  if (shift < 4 || shift > 7) return true;
  const long long page = 1ll << shift;
  return (D != 128 && D != 64) || B < 1 || B > 65534 || N < 0 || M < 1 || H < 1 || H > 65535 || pages < 1 || ldt < M || M * page > 0x7fffff80ll ||
         pages * page * H > 0x7fffff00ll || !k || !v || !starts || !pos || !table || (((uintptr_t)k | (uintptr_t)v) & 31);
}

}  // namespace bones
