// Which row tile and key head a workgroup of k_kv4_rows (kv4.hip) takes. Plain constant expressions, so
// that a host compiler can check that every pair is taken, and once.
#pragma once

namespace spx {

// Place i of n in an order that runs backwards in every other `turn`.
constexpr int snake(int i, int n, int turn) {
  const int b = i / turn * turn, left = n - b < turn ? n - b : turn;
  return i / turn & 1 ? b + left - 1 - (i - b) : i;
}

// The last tiles of a sequence see the most tokens: they go first, about 256 workgroups (one a CU) by
// falling work, as many after them by rising work, and so on. Key heads of a tile are neighbours, and only
// whole tiles change places: a workgroup's head and its tile's place are two parts of one number, whatever
// the number of heads.
struct RowsPlace { int job, head; };
constexpr RowsPlace rows_place(int block, int blocks, int n_kv) {
  const int jobs = blocks / n_kv, turn = n_kv < 256 ? 256 / n_kv : 1;
  return {jobs - 1 - snake(block / n_kv, jobs, turn), block % n_kv};
}

}  // namespace spx
