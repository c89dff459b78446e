// How rows of logits are cut into parts, and what comes before a token, shared
// by host, kernels and plain C++ (the CPU tests compile this file alone).
#pragma once
#if defined(__HIP__) || defined(__HIPCC__)
#define LP_FN __host__ __device__ __forceinline__
#else
#define LP_FN static inline
#endif

// Threads of a workgroup, logits that each takes in a turn of the loop; parts of a row at most; workgroups of a launch
// that has more than one a row, at most.
#define LP_THREADS 256
#define LP_LOGITS 16
#define LP_SPLITS 64
#define LP_WORKGROUPS 768

typedef struct {
  int n;              // parts of a row
  int vecs;           // 16-byte pieces of a part; the last one takes what is left, up to half a turn more
} lp_split;

LP_FN int lp_min(int a, int b) { return a < b ? a : b; }
LP_FN int lp_max(int a, int b) { return a > b ? a : b; }
LP_FN int lp_parts(int pieces, int vecs) { return lp_max(1, (pieces + vecs - 1) / vecs); }

// `rows` rows of V logits, E of them in a piece.  Three workgroups a CU together (96 rows of bf16, top 20: 38 us; two or four
// a CU 40 to 44: a wave's first list costs it 1 us), but two turns of the loop each (one f32 row: 31 parts 19 us, 61 parts
// 21, the join taking longer), in whole turns, the number nearest to that; no part for less than half a turn, which goes
// piece by piece, and no second round of workgroups for a few.
LP_FN lp_split lp_divide(int rows, int V, int E) {
  const int turn = LP_THREADS * LP_LOGITS / E, pieces = V / E;
  const int room = lp_max(1, lp_min(LP_SPLITS, LP_WORKGROUPS / lp_max(rows, 1))), most = lp_max(1, lp_min(room, V / 8192));
  lp_split s;
  if (most == 1) {
    s.n = 1;
    s.vecs = lp_max(pieces, 1);
    return s;
  }
  s.vecs = lp_max(1, (pieces + most * turn / 2) / (most * turn)) * turn;
  s.n = lp_parts(pieces, s.vecs);
  if (s.n > room) {
    s.vecs = (pieces + room * turn - 1) / (room * turn) * turn;
    s.n = lp_parts(pieces, s.vecs);
  }
  if (s.n > 1 && pieces - (s.n - 1) * s.vecs < turn / 2) --s.n;
  return s;
}

// The piece that token `tok` lies in, where pieces of E logits begin behind `head` logits; -1 for one in front of them (or none).
LP_FN int lp_piece(int tok, int head, int E) { return tok < head ? -1 : (tok - head) / E; }
// The bits of the next f32 above one that is a number below +inf.
LP_FN unsigned lp_above(unsigned bits) { return (bits & 0x7fffffffu) == 0 ? 1 : bits & 0x80000000u ? bits - 1 : bits + 1; }
