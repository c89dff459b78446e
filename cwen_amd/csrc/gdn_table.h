// Arithmetic of packed sequences and pool slots, shared by the kernels and plain
// C++ (the CPU tests compile this file alone).  All of it takes what lies in
// memory as it is and yields indexes that are safe to use.
#pragma once
#include <stdbool.h>
#include <stdint.h>
#if defined(__HIP__) || defined(__HIPCC__)
#define GDN_FN __host__ __device__ __forceinline__
#else
#define GDN_FN static inline
#endif

// A border as a row index.
GDN_FN int gdn_border(int cu, int total) { return cu < 0 ? 0 : cu < total ? cu : total; }
// Rows between two borders.
GDN_FN int gdn_rows(int first, int end) { return end > first ? end - first : 0; }
// Whether a sequence of `rows` rows may take `count` of them.
GDN_FN bool gdn_count_ok(int count, int rows) { return count >= 0 && count <= rows; }
// Whether a slot may be read or written; -1 stands for none.
GDN_FN bool gdn_slot_ok(int slot, int n_slots) { return slot >= -1 && slot < n_slots; }
// Whether a sequence that ends in `dst` may not, for what another one names.
GDN_FN bool gdn_clash(int dst, int other_src, int other_dst) { return dst >= 0 && (other_dst == dst || other_src == dst); }
// Sequences cut into pieces of N rows: the first piece of sequence s, whose rows begin at
// `first`.  A sequence's pieces end before the next one's first, so that pieces need
// no sums over the sequences; some numbers are no piece.
GDN_FN int gdn_piece0(int first, int s, int N) { return first / N + s; }
// Pieces of all sequences at most.
GDN_FN long long gdn_pieces(int total, int n_seq, int N) { return (long long)total / N + n_seq; }
