// Sequences of a batch and their pieces, for the operators that keep a state per sequence.
//
// A batch is S sequences of L rows each (row s L + t), or packed rows with offsets cu
// (S + 1): sequence s owns rows [cu[s], cu[s+1]); rows in front of cu[0] and from cu[S] on
// belong to none.
// Every sequence is cut into pieces of Q rows; piece j of the batch is piece k = j - base(s)
// of sequence s with base(s) = s ceil(L / Q), or cu[s] / Q + s for packed rows (rounded
// down): consecutive bases are at least ceil(len / Q) apart, so the pieces of two sequences
// never share an index and floor(T / Q) + S indices hold them all without a table. Offsets
// are clamped to the rows and to one another, so a bad cu gives wrong rows but no access
// outside them.
//
// Slots: sequence s keeps its state in entry slots[s] of a pool (entry s without slots). A
// negative slot means no entry: the sequence starts from zeros and leaves nothing. A slot
// behind the pool, or one that an earlier sequence of the batch has, is refused for that
// sequence: its outputs are NaN and its entry is not touched. fresh[s] != 0: the
// sequence starts from zeros whatever its entry holds.
#pragma once

#include "semx_common.cuh"

namespace semx {

struct SeqMap {
  const int32_t* cu;  // NULL: equal lengths
  int64_t S, T, L;
  int64_t Q, per, pieces;
  const int32_t* slots;
  const uint8_t* fresh;
  int64_t n_slots;  // 0: no pool
};

struct Piece {
  int64_t s, row0;   // sequence and its first row
  int len, t0, t1;   // its length and this piece's steps [t0, t1)
  int k;             // number of the piece in its sequence
  bool live;         // false: no such piece. A sequence without rows has piece 0.
};

// First row of sequence s, and the index of its first piece of Q rows.
__device__ __forceinline__ int64_t seq_start(const SeqMap& m, int64_t s) {
  return m.cu == nullptr ? s * m.L : min(max((int64_t)m.cu[s], (int64_t)0), m.T);
}
__device__ __forceinline__ int64_t piece_base(const SeqMap& m, int64_t s, int64_t Q) {
  return m.cu == nullptr ? s * ((m.L + Q - 1) / Q) : seq_start(m, s) / Q + s;
}

// Piece j. All lanes of the warp call it with the same j (the search over the offsets is
// 32-way: two rounds up to 1024 sequences).
__device__ __forceinline__ Piece find_piece(const SeqMap& m, int64_t j) {
  Piece q;
  q.live = j < m.pieces && m.S > 0;
  if (!q.live) {
    q.s = q.row0 = 0;
    q.len = q.t0 = q.t1 = q.k = 0;
    return q;
  }
  int64_t k;
  if (m.cu == nullptr) {
    q.s = j / m.per;
    k = j - q.s * m.per;
    q.row0 = q.s * m.L;
    q.len = (int)m.L;
  } else {
    int64_t lo = 0, n = m.S;
    const int lane = threadIdx.x & 31;
    while (n > 1) {
      const int64_t step = (n + 31) / 32;
      const int64_t at = lo + lane * step;
      const bool ok = lane * step < n && piece_base(m, at, m.Q) <= j;
      const unsigned hit = __ballot_sync(0xffffffffu, ok);
      const int64_t w = hit == 0u ? 0 : 31 - __clz((int)hit);
      lo += w * step;
      n = min(step, n - w * step);
    }
    q.s = lo;
    q.row0 = seq_start(m, lo);
    q.len = (int)(max(seq_start(m, lo + 1), q.row0) - q.row0);
    k = j - piece_base(m, lo, m.Q);
  }
  q.live = k >= 0 && (k == 0 || k * m.Q < q.len);
  q.k = (int)k;
  q.t0 = q.live ? (int)(k * m.Q) : 0;
  q.t1 = q.live ? (int)min((int64_t)q.len, k * m.Q + m.Q) : 0;
  return q;
}

// First row of the first sequence, and first row behind the last one.
__device__ __forceinline__ int64_t rows_begin(const SeqMap& m) {
  return m.S > 0 && m.cu != nullptr ? seq_start(m, 0) : 0;
}
__device__ __forceinline__ int64_t rows_end(const SeqMap& m) {
  return m.S > 0 ? (m.cu == nullptr ? m.S * m.L : seq_start(m, m.S)) : 0;
}

// Calls f(row) for every pieces-th of the rows that belong to no sequence, from number j on: those
// in front of the first sequence, then those behind the last.
template <class F>
__device__ __forceinline__ void for_unused_rows(const SeqMap& m, int64_t j, F f) {
  const int64_t front = rows_begin(m), count = front + m.T - rows_end(m);
  for (int64_t i = j; i < count; i += m.pieces) f(i < front ? i : m.T - count + i);
}

// Entry of sequence s in the pool: >= 0, or kNone (no entry), or kRefused. Called by all
// threads of the CTA (one barrier).
constexpr int64_t kNone = -1, kRefused = -2;
__device__ __forceinline__ int64_t find_slot(const SeqMap& m, int64_t s) {
  if (m.n_slots == 0) return kNone;
  if (m.slots == nullptr) return s < m.n_slots ? s : kRefused;
  const int32_t mine = m.slots[s];
  int twice = 0;
  if (mine >= 0)
    for (int64_t i = threadIdx.x; i < s; i += blockDim.x) twice |= m.slots[i] == mine;
  twice = __syncthreads_or(twice);
  if (mine < 0) return kNone;
  return twice || mine >= m.n_slots ? kRefused : mine;
}

// Entries of sequences [s0, s0 + n), n at most RUN <= blockDim.x, into out (shared memory). Called by
// all threads of the CTA; ends with a barrier.
template <int RUN>
__device__ __forceinline__ void find_slots(const SeqMap& m, int64_t s0, int n, int64_t* out) {
  const int tid = threadIdx.x;
  if (m.n_slots == 0 || m.slots == nullptr) {
    if (tid < n) out[tid] = m.n_slots == 0 ? kNone : s0 + tid < m.n_slots ? s0 + tid : kRefused;
    __syncthreads();
    return;
  }
  __shared__ int32_t run[RUN];
  if (tid < n) {
    const int32_t mine = m.slots[s0 + tid];
    run[tid] = mine;
    out[tid] = mine < 0 ? kNone : mine >= m.n_slots ? kRefused : mine;
  }
  __syncthreads();
  // Every earlier slot against the run's. Threads that find a pair write the same value.
  for (int64_t i = tid; i < s0 + n; i += blockDim.x) {
    const int32_t v = m.slots[i];
    for (int k = (int)max((int64_t)0, i - s0 + 1); k < n; ++k)
      if (v >= 0 && run[k] == v) out[k] = kRefused;
  }
  __syncthreads();
}

// Host: fills the sequence fields for pieces of Q rows (Q <= 0: one piece per sequence).
inline void set_pieces(SeqMap* m, int64_t Q) {
  if (Q <= 0) Q = (int64_t)1 << 31;  // longer than any sequence
  m->Q = Q;
  m->per = m->L > 0 ? cdiv(m->L, Q) : 1;
  m->pieces = m->cu == nullptr ? m->S * m->per : m->T / Q + m->S;
}

// Host: a forward without rows and without a pool has no output. It returns before it looks for its
// GPU, which only an output's address could tell.
inline bool nothing_to_do(const SeqMap& m) { return m.T == 0 && (m.S == 0 || m.n_slots == 0); }

// Host: checks the sequence fields shared by the argument structs.
inline int check_seqs(const char* what, int64_t S, int64_t T, int64_t L, const int32_t* cu, const void* state,
                      const int32_t* slots, const uint8_t* fresh, int64_t n_slots, SeqMap* m) {
  if (S < 0 || T < 0 || L < 0 || n_slots < 0)
    return fail(SEMX_ERR_SHAPE, "%s: S=%lld, rows=%lld, L=%lld, n_slots=%lld", what, (long long)S, (long long)T,
                (long long)L, (long long)n_slots);
  if (S >= ((int64_t)1 << 31) - 1 || T >= ((int64_t)1 << 31) - 1 || L >= ((int64_t)1 << 31) - 1)
    return fail(SEMX_ERR_SHAPE, "%s: S=%lld, rows=%lld, L=%lld", what, (long long)S, (long long)T, (long long)L);
  if (cu == nullptr && S * L != T)
    return fail(SEMX_ERR_SHAPE, "%s: %lld sequences of %lld rows are not %lld rows", what, (long long)S, (long long)L,
                (long long)T);
  if ((state != nullptr) != (n_slots > 0))
    return fail(SEMX_ERR_NULL, "%s: a state needs entries, and entries a state", what);
  if (state == nullptr && (slots != nullptr || fresh != nullptr))
    return fail(SEMX_ERR_NULL, "%s: slots / fresh without a state", what);
  if (state != nullptr && slots == nullptr && n_slots < S)
    return fail(SEMX_ERR_SHAPE, "%s: %lld entries for %lld sequences", what, (long long)n_slots, (long long)S);
  *m = SeqMap{cu, S, T, L, 0, 0, 0, slots, fresh, n_slots};
  return SEMX_OK;
}

}  // namespace semx
