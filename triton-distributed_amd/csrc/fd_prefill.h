// Attention of many query rows over packed keys or over the paged cache (gfx950): prompts, chunks of prompts, drafted
// tokens, and the prefix part of a shared-prefix decode step.
//
// out[i,h] = sum_j softmax_j(scale q[i,h].k[j,h/G]) v[j,h/G] over the keys j that row i sees: j < n_k, and in the causal
// form j <= i + n_k - n_q (the last query sees the last key; a length beyond the table's room counts in full here).  One pass over the keys with the running maximum m and sum
// l of the softmax; the accumulator is rescaled only when the maximum has grown by more than 2^8 (as in
// fd_softmax_step).
//
// Rows: the G query heads of a KV head share its keys, so a row is a (token, head of the group) pair, r = token * G + head,
// and a tile owns consecutive rows of one sequence and one KV head: a causal tile of G = 4 spans a quarter of the tokens that
// as many rows of one head would, and wastes that much less on its diagonal.
// Both products run on v_mfma_f32_32x32x16 with the scores transposed, S^T[token][row] = K Q^T and
// O^T[dim][row] += V^T P^T: lane l then holds scores of row l % 32 only -- 16 of the 32 tokens of a block, tokens
// 8 (i / 4) + 4 (l / 32) + i % 4 -- so a row's maximum and sum are in-lane reductions plus one exchange between the wave
// halves, and those tokens are, eight at a time, exactly the k indices that the lane supplies as B operand of the second
// product: P never leaves its registers.  V comes from LDS through the transposing read (ds_read_b64_tr_b16): 16 lanes
// read four tokens of 16 dims and receive four tokens of one dim each.
// Keys go global -> LDS without passing through registers (16-bit caches; 16 bytes a lane).  The LDS image of such a load is
// lane-linear, so rows are swizzled at the source: lane c of a row fetches the 16-byte chunk c ^ f(row), with f chosen so that
// the 128-bit K reads (32 rows of one chunk column) and the transposing V reads (8 rows of 64 bytes) both touch all 64 banks
// (no bank conflicts counted).  An fp8 cache is converted on its way to LDS (exact) instead.
//
// Two ways to share the work of a tile among the four waves of a workgroup:
//  * rows (fd_row_tile): 128 rows, 32 a wave, all waves on the same 64 keys, which are two tiles deep in LDS.  Bound: the
//    matrix pipes, then power -- one prompt of 16384 tokens, 32/8 heads of 128, bf16: 2.1 ms = 1.05 PFLOP/s at a clock that
//    the chip lowers to 1.7 GHz (an 8192^3 library product in the same session: 1.22 PFLOP/s).
//  * keys (fd_key_tile): 32 rows, all waves on the same rows, every wave on 32 keys of its own at a time, in its own part of
//    LDS, without a barrier until their states are joined at the end.  Bound: HBM -- eight sequences of 8000 tokens with five
//    drafted tokens each, 32/8 heads of 128, bf16: 45 us = 5.8 TB/s and 4.6 us for the merge of their key ranges.
//
// Tokens past a sequence's length are never fetched: the row address is clamped to the last token, and what such a row
// holds is masked.  A masked score has weight 0, and 0 times a V row that is finite is 0; a V row that holds an infinity
// or NaN would turn rows that do not see it into NaN, so work whose result is not finite is done once more with the
// non-finite V values taken out of the masked tiles' products and added to the rows that see them only.
#pragma once

#include "fd_mma.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

// The query rows of sequence b: `count` tokens from `start` on (whatever cu_q holds, inside [0, total_q)).  Without cu_q
// there is one sequence, all rows.
__device__ __forceinline__ void fd_prefill_span(const PrefillArgs& a, int b, int& start, int& count) {
  start = 0;
  count = a.total_q;
  if (a.cu_q) {
    start = min(max(a.cu_q[b], 0), a.total_q);
    count = min(max(a.cu_q[b + 1], start), a.total_q) - start;
  }
  if (a.q_lens) count = min(count, max(a.q_lens[b], 0));
}

namespace {

template <typename T>
struct Mma32;
template <>
struct Mma32<__bf16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  }
  static constexpr uint32_t kExp = 0x7f807f80u;   // exponent bits of both halves
};
template <>
struct Mma32<_Float16> {
  static __device__ __forceinline__ f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
  }
  static constexpr uint32_t kExp = 0x7c007c00u;
};

// v and the other half's value of the same row
__device__ __forceinline__ float half_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// 16 bytes per lane from global memory to lds_base + 16 * lane.  Inline assembly, so that the compiler does not put a wait
// for it in front of the LDS reads of the other buffer; the kernel waits itself (vmcnt(0)) before the barrier that
// publishes the tile.  The instruction has no register output.
// STREAM: past the caches, for rows that are read once.
template <bool STREAM>
__device__ __forceinline__ void load_to_lds_b128(const void* src, uint32_t lds_base) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds_base), "v"(src)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_base), "v"(src)
                 : "memory", "m0");
}

__device__ __forceinline__ u32x4 lds_read_b128(const char* p) { return *(const u32x4*)p; }

__device__ __forceinline__ u32x2 lds_read_tr(const char* p) {
  typedef __attribute__((address_space(3))) i16x4* lds_ptr;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(i16x4*)p));
}

template <int D>
struct PrefillTile {
  static constexpr int kRowB = 2 * D;          // bytes of a 16-bit row in LDS
  static constexpr int kChunks = D / 8;        // 16-byte chunks of it
  // chunk c of row r lies at position c ^ k_swz(r) / c ^ v_swz(r) of the row
  static __device__ __forceinline__ int k_swz(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int v_swz(int r) { return D == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2; }
};

// A unit of work: 32- or 128-row tile j of a sequence's rows (q_start, n_q tokens of G rows) for one KV head, and range `split`
// of its keys.
struct PrefillItem {
  int kvh, q_start, n_q, j, k_start, n_k, slot, split, splits, min_tiles, causal;
  int ahead;                 // causal: token i of the rows stands behind i + ahead keys
  const int32_t* table;      // nullptr: packed keys from k_start on

  // keys that row r of the sequence sees: [0, limit_of(r))
  __device__ __forceinline__ int token_of(const PrefillArgs& a, int r) const {
    return (int)(((uint64_t)(uint32_t)r * a.g_magic) >> a.g_shift);
  }
  __device__ __forceinline__ int limit_of(const PrefillArgs& a, int r) const {
    return causal ? min(n_k, token_of(a, r) + 1 + ahead) : n_k;
  }
  // The token row of the pool that holds key `tok` (any value: keys past the last one repeat it); `entry`: its page, so that
  // the table can be read ahead of its use.
  __device__ __forceinline__ int page_entry(const PrefillArgs& a, int tok) const {
    if (!table) return 0;
    return table[((uint64_t)(uint32_t)min(tok, n_k - 1) * a.p_magic) >> a.p_shift];
  }
  __device__ __forceinline__ int pool_row(const PrefillArgs& a, int tok, int entry) const {
    tok = min(tok, n_k - 1);
    if (!table) return k_start + tok;
    const int pg = (int)(((uint64_t)(uint32_t)tok * a.p_magic) >> a.p_shift);
    return min(max(entry, 0), a.num_pages - 1) * a.P + (tok - pg * a.P);
  }
};

// Among up to 64 sequences, one a lane: the tiles of those that come before this lane's -- longest first -- and of all.
__device__ __forceinline__ int fd_tiles_before(int keys, int tiles, int n, int* total) {
  const int lane = threadIdx.x & 63;
  int before = 0, all = 0;
  for (int i = 0; i < n; ++i) {
    const int k_i = __builtin_amdgcn_readlane(keys, i), t_i = __builtin_amdgcn_readlane(tiles, i);
    before += k_i > keys || (k_i == keys && i < lane) ? t_i : 0;
    all += t_i;
  }
  *total = all;
  return before;
}

// Steps over blocks of 64 K sequences from b0 on that end before row tile `tile` of the list; `base`: the tiles before b0.
template <int K>
__device__ __forceinline__ void fd_skip_sequences(const PrefillArgs& a, int bm, int tile, int& b0, int& base) {
  const int lane = threadIdx.x & 63;
  while (b0 < a.batch) {
    int total = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int b = b0 + lane * K + k;
      int start, count = 0;
      if (b < a.batch) fd_prefill_span(a, b, start, count);
      total += (count * a.G + bm - 1) / bm;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off);
    total = __builtin_amdgcn_readfirstlane(total);
    if (tile - base < total) return;
    base += total;
    b0 += 64 * K;
  }
}

// The lane whose `keys` (at most `top`) are the rank-th largest of the wave's, equal ones in the order of their lanes: the
// value bit by bit from above, then the lane among those that hold it.
__device__ __forceinline__ int fd_lane_of_rank(int keys, int rank, int top) {
  int value = 0;
  for (int bit = 31 - __builtin_clz(top | 1); bit >= 0; --bit) {
    const int with = value | 1 << bit;
    if (__popcll(__ballot(keys >= with)) > rank) value = with;
  }
  const uint64_t equal = __ballot(keys == value);
  const int at = rank - __popcll(__ballot(keys > value));
  const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(equal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)equal, 0));
  return __builtin_ctzll(__ballot(keys == value && before == at));
}

// The unit of this workgroup: KV head fastest (the eight XCDs take neighbouring workgroups in turn, so with eight KV heads
// each XCD's L2 holds one head's keys), then the key range, then the row tile.  own: one of a shared-prefix step's sequences
// with its own keys (tiles of 32 rows).  Those units, which are bound by memory, and the groups', which are bound by the
// matrix pipes, are dealt out a chip's worth at a time in turn, so that a CU holds one of each (64 sequences behind 8192
// tokens 46 -> 39 us, four groups over fp8 142 -> 126 us against all of the groups' first, both as they were then).  false: no
// such unit.
__device__ __forceinline__ bool fd_find_item(const PrefillArgs& a, int bm, PrefillItem& it, bool& own) {
  const int lane = threadIdx.x & 63;
  uint32_t at = blockIdx.x;
  own = false;
  if (a.own_splits > 0) {
    constexpr uint32_t kDeal = 256;
    const uint32_t n_group = (uint32_t)a.group_units * a.Hkv, n_own = (uint32_t)a.own_units * a.Hkv;
    const uint32_t dealt = (n_group < n_own ? n_group : n_own) / kDeal * kDeal;
    if (at < 2 * dealt) {
      own = at % (2 * kDeal) >= kDeal;
      at = at / (2 * kDeal) * kDeal + at % kDeal;
    } else {
      at -= dealt;
      own = at >= n_group;
      if (own) at -= n_group - dealt;
    }
  }
  it.kvh = at % a.Hkv;
  int unit = at / a.Hkv;
  it.k_start = 0;
  if (own) {
    it.splits = a.own_splits;
    it.min_tiles = a.own_min_tiles;
    it.split = unit % it.splits;
    it.slot = a.splits + it.split;
    const int rest = unit / it.splits, tiles = (a.G + 31) / 32;
    const int place = rest / tiles;           // longest first within 64 sequences
    it.j = rest - place * tiles;
    if (place >= a.total_q) return false;
    const int b0 = place & ~63, n = min(64, a.total_q - b0);
    const int keys = lane < n ? min(max(a.own_lens[b0 + lane], 0), a.own_max_pages * a.P) : -1;
    const int w = fd_lane_of_rank(keys, place - b0, a.own_max_pages * a.P);
    it.q_start = b0 + w;
    it.n_k = __builtin_amdgcn_readlane(keys, w);
    it.n_q = 1;
    it.causal = it.ahead = 0;
    it.table = a.own_bt + (int64_t)it.q_start * a.own_sbt;
    return true;
  }
  it.splits = a.splits;
  it.min_tiles = a.min_tiles;
  it.split = it.slot = unit % it.splits;
  it.causal = a.causal;
  const int tile = unit / it.splits;
  // The row tile of the list: sequences with the most keys first (in blocks of 64 sequences, one a lane), the tiles of a
  // sequence from its end, where a causal row sees the most -- short work fills in behind long.  Every workgroup looks for its
  // own: large batches are stepped through in blocks of 512 and 64 (one token on each of 512 / 5000 caches of up to 400
  // tokens, 32/8 heads of 128: 328 us / 21.7 ms with the loop over a block's lanes below in every block, 151 us / 1.9 ms).
  int b0 = 0, base = 0;
  if (a.batch > 64) {
    fd_skip_sequences<8>(a, bm, tile, b0, base);
    fd_skip_sequences<1>(a, bm, tile, b0, base);
  }
  for (; b0 < a.batch; b0 += 64) {
    const int mine = b0 + lane;
    int qs = 0, nq = 0, ks = 0, nk = -1, length = 0, tiles = 0;
    if (mine < a.batch) {
      fd_prefill_span(a, mine, qs, nq);
      if (a.bt) {
        length = max(a.kv_lens[mine], 0);         // what the table has no room for counts for the rows' places
        nk = min(length, a.max_pages * a.P);
      } else {
        ks = min(max(a.cu_k[mine], 0), a.total_k);
        nk = length = min(max(a.cu_k[mine + 1], ks), a.total_k) - ks;
      }
      tiles = (nq * a.G + bm - 1) / bm;
    }
    int total;
    const int place = tile - base - fd_tiles_before(nk, tiles, min(64, a.batch - b0), &total);
    const uint64_t here = __ballot(place >= 0 && place < tiles);
    if (here) {
      const int w = __builtin_ctzll(here);
      it.q_start = __builtin_amdgcn_readlane(qs, w);
      it.n_q = __builtin_amdgcn_readlane(nq, w);
      it.k_start = __builtin_amdgcn_readlane(ks, w);
      it.n_k = __builtin_amdgcn_readlane(nk, w);
      it.ahead = __builtin_amdgcn_readlane(length, w) - it.n_q;
      it.j = __builtin_amdgcn_readlane(tiles, w) - 1 - __builtin_amdgcn_readlane(place, w);
      it.table = a.bt ? a.bt + (int64_t)(b0 + w) * a.sbt : nullptr;
      return true;
    }
    base += total;
  }
  return false;
}

// What both bodies share: a wave's 32 rows, its 32-key blocks, its softmax state.
template <typename T, bool FP8, bool CAP, int D>
struct PrefillWave {
  using Tile = PrefillTile<D>;
  static constexpr int KS = D / 16;            // k steps of the scores
  static constexpr int MB = D / 32;            // dim blocks of the output
  static constexpr int kInChunks = FP8 ? D / 16 : Tile::kChunks;   // 16-byte chunks of a row in memory

  const PrefillArgs& a;
  const PrefillItem& it;
  int lane, half, l32;
  int q_tok, q_head, my_limit, lo_limit;       // of this lane's row; keys that all rows of the wave see
  bool real_row;
  u32x4 qf[KS];
  float c, cap, cap_in;
  int k_lane, v_lane, v_swz;
  const char* kb;
  const char* vb;
  uint32_t sk_b, sv_b;
  f32x16 o[MB];
  float m, l;

  // row0: first of the wave's rows
  __device__ __forceinline__ PrefillWave(const PrefillArgs& args, const PrefillItem& item, int row0)
      : a(args), it(item), lane(threadIdx.x & 63), half(lane >> 5), l32(lane & 31) {
    const int rows = it.n_q * a.G;
    const int row = min(row0 + l32, rows - 1);   // rows past the end repeat the last one and are not stored
    real_row = row0 + l32 < rows;
    q_tok = it.token_of(a, row);
    q_head = row - q_tok * a.G;
    my_limit = it.limit_of(a, row);
    lo_limit = it.limit_of(a, min(row0, rows - 1));
    // Q^T as B operand: lane (row, half) holds dims 16 ks + 8 half .. + 7
    const char* qp = (const char*)a.q + 2 * ((int64_t)(it.q_start + q_tok) * a.sq_t + (int64_t)(it.kvh * a.G + q_head) * a.sq_h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const u32x4*)(qp + 32 * ks + 16 * half);
    c = a.sm_scale;
    if (FP8) c *= a.k_scale[it.kvh];
    cap = cap_in = 0.f;
    if constexpr (CAP) {            // x = cap tanh(s c / cap), in the base-2 domain afterwards
      cap_in = 2.0f * FD_LOG2E * c / a.soft_cap;
      cap = a.soft_cap * FD_LOG2E;
      c = 1.f;
    } else {
      // the maximum is taken over the raw scores, so the factor has to be positive: a negative one goes into Q (exact)
      if (c < 0.f) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] ^= 0x80008000u;
      }
      c = fmaxf(fabsf(c) * FD_LOG2E, 1e-30f);
    }
    k_lane = l32 * Tile::kRowB + ((half ^ Tile::k_swz(l32)) << 4);   // rows of a K read: l32 + a multiple of 32
    const int vi = lane & 15, v_tok = 4 * half + (vi >> 2);
    v_lane = v_tok * Tile::kRowB + ((lane >> 4) & 1) * 32 + (vi & 3) * 8;
    v_swz = Tile::v_swz(v_tok) << 4;             // the same for all token steps of 8
    kb = (const char*)a.k + (FP8 ? 1 : 2) * ((int64_t)it.kvh * a.sk_h);
    vb = (const char*)a.v + (FP8 ? 1 : 2) * ((int64_t)it.kvh * a.sv_h);
    // (a pool has fewer than 2^31 rows and a row stride fits 32 bits: one 32 x 32 -> 64 bit multiply an address)
    sk_b = (uint32_t)a.sk_t * (FP8 ? 1 : 2);
    sv_b = (uint32_t)a.sv_t * (FP8 ? 1 : 2);
  }

  __device__ __forceinline__ void start() {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) o[mb] = f32x16{};
    m = -3.0e38f;     // below every score: a row that sees nothing keeps l = 0
    l = 0.f;
  }

  // A fragment of K (rows 32 tb .. + 31 of the tile at `tile`, k step ks) and of V^T (token step st, dim block mb).
  __device__ __forceinline__ u32x4 k_frag(const char* tile, int ks, int tb) const {
    return lds_read_b128(tile + (k_lane ^ (ks << 5)) + tb * 32 * Tile::kRowB);
  }
  __device__ __forceinline__ u32x4 v_frag(const char* tile, int st, int mb) const {
    const char* vp = tile + v_lane + st * 16 * Tile::kRowB + ((mb << 6) ^ v_swz);
    const u32x2 lo = lds_read_tr(vp), hi = lds_read_tr(vp + 8 * Tile::kRowB);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }

  // Where chunk ch of row r of a K (V) tile comes from, relative to the row, and where its 16-bit form lies in the tile.
  static __device__ __forceinline__ int source_chunk(bool is_k, int r, int ch) {
    return FP8 ? ch : ch ^ (is_k ? Tile::k_swz(r) : Tile::v_swz(r));
  }
  // fp8: 16 values of row r, chunk ch, converted into the tile
  static __device__ __forceinline__ void deposit(bool is_k, char* tile, int r, int ch, u32x4 raw) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x4 x = {Mma<T>::from_fp8(raw[2 * h], false), Mma<T>::from_fp8(raw[2 * h], true),
                       Mma<T>::from_fp8(raw[2 * h + 1], false), Mma<T>::from_fp8(raw[2 * h + 1], true)};
      *(u32x4*)(tile + r * Tile::kRowB + (((2 * ch + h) ^ (is_k ? Tile::k_swz(r) : Tile::v_swz(r))) << 4)) = x;
    }
  }

  // Soft cap and mask of the raw scores of 32 NB keys from t0 on (the mask is a wave-uniform branch that most tiles pass by).
  template <int NB>
  __device__ __forceinline__ void finish_scores(int t0, f32x16 (&s)[NB]) const {
    if constexpr (CAP) {
#pragma unroll
      for (int tb = 0; tb < NB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = fd_exp2(s[tb][i] * cap_in);
          s[tb][i] = __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + e), cap);   // tanh(y) = 1 - 2 / (1 + e^2y)
        }
    }
    if (t0 + 32 * NB > lo_limit) {
      const int see = my_limit - t0 - 4 * half;
#pragma unroll
      for (int tb = 0; tb < NB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[tb][i] = tb * 32 + 8 * (i / 4) + i % 4 < see ? s[tb][i] : -INFINITY;
    }
  }

  // The reference point follows the maximum `mx` of the raw scores that come next (this lane's keys of its row).
  __device__ __forceinline__ void move_reference(float mx) {
    const float top = fmaxf(m, half_max(mx) * c);
    const float m_new = top - m > 8.0f ? top : m;
    if (__any(m_new > m)) {
      const float alpha = fd_exp2(m - m_new);
      l *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[mb] *= alpha;
      m = m_new;
    }
  }

  // One tile without a pipeline: scores, weights, product.  CAREFUL: keeps non-finite V values from rows that do not see them.
  template <int NB, bool CAREFUL, typename F>
  __device__ __forceinline__ void plain_tile(const char* k_tile, const char* v_tile, int t0, F after_scores) {
    f32x16 s[NB];
#pragma unroll
    for (int tb = 0; tb < NB; ++tb) s[tb] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) s[tb] = Mma32<T>::run(k_frag(k_tile, ks, tb), qf[ks], s[tb]);
    after_scores();
    finish_scores(t0, s);
    const bool masked = t0 + 32 * NB > lo_limit;
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e) mx = fmaxf(mx, s[e / 16][e % 16]);
    move_reference(mx);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16 * NB; ++e) {
      s[e / 16][e % 16] = fd_exp2(__builtin_fmaf(s[e / 16][e % 16], c, -m));
      sum += s[e / 16][e % 16];
    }
    l += sum;
#pragma unroll
    for (int st = 0; st < 2 * NB; ++st) {
      u32x4 pf;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        pf[w] = Mma<T>::pack(s[st / 2][8 * (st % 2) + 2 * w], s[st / 2][8 * (st % 2) + 2 * w + 1]);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        u32x4 vf = v_frag(v_tile, st, mb);
        if (CAREFUL && masked) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t e = vf[w] & Mma32<T>::kExp;
            if ((e & 0xffffu) == (Mma32<T>::kExp & 0xffffu)) vf[w] &= 0xffff0000u;
            if ((e >> 16) == (Mma32<T>::kExp >> 16)) vf[w] &= 0xffffu;
          }
        }
        o[mb] = Mma32<T>::run(vf, pf, o[mb]);
      }
    }
    if (!CAREFUL || !masked) return;
    // the non-finite V values of this tile, for the rows that see them: lane (row, half) owns dims 32 mb + 8 i + 4 half .. + 3
    for (int n = 0; n < 32 * NB; ++n) {
      const char* vr = v_tile + n * Tile::kRowB;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d0 = 32 * mb + 8 * i + 4 * half;
          const u32x2 w = *(const u32x2*)(vr + ((((d0 >> 3) ^ Tile::v_swz(n)) << 4) | ((d0 & 4) << 1)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t bits = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            if ((bits & (uint16_t)Mma32<T>::kExp) == (uint16_t)Mma32<T>::kExp && t0 + n < my_limit)
              o[mb][4 * i + e] += (float)__builtin_bit_cast(T, bits);
          }
        }
    }
  }

  __device__ __forceinline__ bool not_finite() const {   // (x - x is 0 for finite x)
    float probe = l - l;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) probe += o[mb][i] - o[mb][i];
    return __any(!(probe == 0.f));
  }

  // l: already summed over the wave halves
  __device__ __forceinline__ void store() {
    if (!real_row) return;
    // a NaN scale: the lower bound of c dropped it (kept apart from the scores, it leaves rows that see nothing as they are)
    const float scale = FP8 ? a.sm_scale * a.k_scale[it.kvh] : a.sm_scale;
    if (scale != scale && my_limit > 0) l = scale;
    float inv = l != 0.f ? 1.0f / l : 0.f;
    const float lse = l != 0.f ? m * FD_LN2 + __logf(l) : -INFINITY;
    if (FP8) inv *= a.v_scale[it.kvh];
    const int64_t tok = it.q_start + q_tok;
    const int head = it.kvh * a.G + q_head;
    if (a.part) {
      const int64_t at = (tok * a.Hq + head) * (a.splits + a.own_splits) + it.slot;
      if (half == 0) a.part_lse[at] = lse;
      if (l == 0.f) return;         // weight 0: the row is not looked at
      float* dst = a.part + at * D;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *(f32x4*)(dst + 32 * mb + 8 * i + 4 * half) =
              f32x4{o[mb][4 * i] * inv, o[mb][4 * i + 1] * inv, o[mb][4 * i + 2] * inv, o[mb][4 * i + 3] * inv};
    } else {
      if (a.lse && half == 0) a.lse[tok * a.Hq + head] = lse;
      char* dst = (char*)a.out + 2 * (tok * a.so_t + (int64_t)head * a.so_h);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x2 w = {Mma<T>::pack(o[mb][4 * i] * inv, o[mb][4 * i + 1] * inv),
                           Mma<T>::pack(o[mb][4 * i + 2] * inv, o[mb][4 * i + 3] * inv)};
          *(u32x2*)(dst + 2 * (32 * mb + 8 * i + 4 * half)) = w;
        }
    }
  }
};

constexpr int kPrefillWaves = 4;
constexpr int kPrefillLds = 65536;             // two workgroups a CU; the reach of the direct loads' 16-bit LDS offset
// Keys of a row tile: K and V, two deep, fill the LDS.  Waves of a key tile: 32 keys of K and V each.
constexpr int row_tile_keys(int D) { return D == 256 ? 32 : 64; }
constexpr int key_tile_waves(int D) { return D == 256 ? 2 : kPrefillWaves; }

// Four waves of 32 rows over the same keys.
template <typename T, bool FP8, bool CAP, int D>
__device__ __forceinline__ void fd_row_tile(const PrefillArgs& a, const PrefillItem& it, char* smem) {
  using W = PrefillWave<T, FP8, CAP, D>;
  using Tile = PrefillTile<D>;
  constexpr int NW = kPrefillWaves, BM = 32 * NW, BN = row_tile_keys(D), NB = BN / 32, KS = W::KS, MB = W::MB;
  constexpr int kTileB = BN * Tile::kRowB;
  constexpr int kLoads = BN * W::kInChunks / (64 * NW);   // loads per lane and operand
  static_assert(4 * kTileB <= kPrefillLds, "[2][K tile, V tile]");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = it.j * BM, rows = it.n_q * a.G;
  W w(a, it, r0 + wave * 32);
  const int lane = w.lane;
  const int all_tiles = (max(it.limit_of(a, min(r0 + BM - 1, rows - 1)), 0) + BN - 1) / BN;
  const int per_split = max((all_tiles + it.splits - 1) / it.splits, it.min_tiles);
  const int t_first = min(it.split * per_split, all_tiles);
  const int t_last = min(t_first + per_split, all_tiles);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  auto k_tile = [&](int buf) { return smem + 2 * buf * kTileB; };
  auto v_tile = [&](int buf) { return smem + (2 * buf + 1) * kTileB; };

  // ---- tile loads: 16-byte chunk n = (i NW + wave) 64 + lane of a tile.  Lane k looks up the row of token k.
  auto page_entry = [&](int t) { return it.page_entry(a, t * BN + min(lane, BN - 1)); };
  int pr[kLoads];                                         // pool rows that this lane fetches from
  u32x4 f8k[FP8 ? kLoads : 1], f8v[FP8 ? kLoads : 1];
  auto rows_of = [&](int t, int entry) {
    const int row = it.pool_row(a, t * BN + min(lane, BN - 1), entry);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) pr[i] = __shfl(row, ((i * NW + wave) * 64 + lane) / W::kInChunks);
  };
  auto request_one = [&](bool is_k, int buf, int i) {
    const int n = (i * NW + wave) * 64 + lane;
    const int r = n / W::kInChunks, ch = n % W::kInChunks;
    const char* src = (is_k ? w.kb : w.vb) + (uint64_t)(uint32_t)pr[i] * (is_k ? w.sk_b : w.sv_b) + (W::source_chunk(is_k, r, ch) << 4);
    if constexpr (FP8)
      (is_k ? f8k : f8v)[i] = *(const u32x4*)src;
    else
      load_to_lds_b128<false>(src, __builtin_amdgcn_readfirstlane(lds0 + (2 * buf + (is_k ? 0 : 1)) * kTileB + (i * NW + wave) * 1024));
  };
  auto request = [&](bool is_k, int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) request_one(is_k, buf, i);
  };
  auto deposit = [&](bool is_k, int buf) {   // fp8: convert what `request` fetched and put it into LDS
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int n = (i * NW + wave) * 64 + lane;
        W::deposit(is_k, is_k ? k_tile(buf) : v_tile(buf), n / W::kInChunks, n % W::kInChunks, (is_k ? f8k : f8v)[i]);
      }
    }
  };
  auto publish = [&] {   // what was requested is in LDS, for every wave, and nobody reads what is requested next
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // One tile of the pipelined walk.  On entry `cur` holds tile t's finished scores, which the reference point has followed,
  // pr the pool rows of tile t + 1, whose K is on its way, like V of tile t.  The scores of tile t + 1 are computed while
  // the weights of tile t are (one MFMA and a few weights at a time: the matrix pipe works on one while the vector pipe
  // does the others), and their maximum while V of tile t is multiplied.
  constexpr int kEvery = KS / 2 / kLoads;  // k steps between two requests
  static_assert(KS == 2 * kEvery * kLoads, "the requests fit under the scores");
  constexpr int E = 16 * NB;               // scores of a lane
  auto step = [&](int t, int& entry, f32x16 (&cur)[NB], f32x16 (&nxt)[NB], auto next_tag) {
    constexpr bool NEXT = decltype(next_tag)::value;
    const int buf = (t - t_first) & 1;
    publish();
    // P is rounded to the query's type for the second product (the sum l is not): half a step, 2^-8 (bf16) or 2^-11 (fp16)
    // of each weight, of both signs -- less in their sum than the rounding of the output itself
    u32x4 pf[BN / 16];
    float sum0 = 0.f, sum1 = 0.f;
    auto weights = [&](int e0, int e1) {   // scores e0 .. e1 - 1, in pairs
#pragma unroll
      for (int e = e0; e < e1; e += 2) {
        const float p0 = fd_exp2(__builtin_fmaf(cur[e / 16][e % 16], w.c, -w.m));
        const float p1 = fd_exp2(__builtin_fmaf(cur[e / 16][e % 16 + 1], w.c, -w.m));
        sum0 += p0;
        sum1 += p1;
        pf[e / 8][e % 8 / 2] = Mma<T>::pack(p0, p1);
      }
    };
    if constexpr (NEXT) {
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) nxt[tb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) nxt[tb] = Mma32<T>::run(w.k_frag(k_tile(buf ^ 1), ks, tb), w.qf[ks], nxt[tb]);
        weights(E * ks / KS & ~1, E * (ks + 1) / KS & ~1);
        // the next requests, one at a time under the MFMAs: V of t + 1 over V of t - 1, then K of t + 2 over K of t (past the
        // end of the range the last key's, which nobody reads: a branch here would cut the block that the compiler schedules)
        if (ks < KS / 2) {
          if (ks % kEvery == 0) request_one(false, buf ^ 1, ks / kEvery);
        } else {
          if (ks == KS / 2) rows_of(t + 2, entry);
          if (ks % kEvery == 0) request_one(true, buf, (ks - KS / 2) / kEvery);
        }
      }
      // pinned here: left to itself the compiler moves the weights behind the branches of finish_scores, next to their use
#pragma unroll
      for (int st = 0; st < BN / 16; ++st) asm volatile("" : "+v"(pf[st]));
      w.l += sum0 + sum1;
      asm volatile("" : "+v"(w.l));
      w.finish_scores((t + 1) * BN, nxt);
    } else {
      weights(0, E);
      w.l += sum0 + sum1;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < BN / 16; ++st)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        w.o[mb] = Mma32<T>::run(w.v_frag(v_tile(buf), st, mb), pf[st], w.o[mb]);
        if constexpr (NEXT) {
          constexpr int N = BN / 16 * MB;  // MFMAs of this product
          const int at = st * MB + mb;
#pragma unroll
          for (int e = E * at / N; e < E * (at + 1) / N; ++e) mx = fmaxf(mx, nxt[e / 16][e % 16]);
        }
      }
    if constexpr (NEXT) {
      w.move_reference(mx);                // (before the barrier, where the wave waits anyway)
      deposit(false, buf ^ 1);
      deposit(true, buf);
      entry = page_entry(t + 3);
    }
  };

  // The walk: K of the first two tiles and V of the first are requested, the scores of the first computed, then a step a
  // tile.  ACTIVE: a wave whose rows are all past the end only fetches.
  auto walk = [&](auto active_tag) {
    constexpr bool ACTIVE = decltype(active_tag)::value;
    w.start();
    if (t_first >= t_last) return;
    rows_of(t_first, page_entry(t_first));
    int entry = page_entry(t_first + 1);
    request(true, 0);
    request(false, 0);
    deposit(true, 0);
    deposit(false, 0);
    publish();
    if (t_first + 1 < t_last) {
      rows_of(t_first + 1, entry);
      entry = page_entry(t_first + 2);
      request(true, 1);
    }
    if constexpr (ACTIVE) {
      f32x16 s0[NB], s1[NB];
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) s0[tb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) s0[tb] = Mma32<T>::run(w.k_frag(k_tile(0), ks, tb), w.qf[ks], s0[tb]);
      w.finish_scores(t_first * BN, s0);
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) mx = fmaxf(mx, s0[e / 16][e % 16]);
      w.move_reference(mx);
      if (t_first + 1 < t_last) deposit(true, 1);
      int t = t_first;
      for (; t + 2 < t_last; t += 2) {       // two tiles a turn: the two sets of scores change places without copies
        step(t, entry, s0, s1, std::true_type{});
        step(t + 1, entry, s1, s0, std::true_type{});
      }
      if (t + 1 < t_last) {
        step(t, entry, s0, s1, std::true_type{});
        step(t + 1, entry, s1, s0, std::false_type{});
      } else {
        step(t, entry, s0, s1, std::false_type{});
      }
    } else {
      if (t_first + 1 < t_last) deposit(true, 1);
      for (int t = t_first; t < t_last; ++t) {
        const int buf = (t - t_first) & 1;
        publish();
        if (t + 1 >= t_last) continue;
        request(false, buf ^ 1);
        rows_of(t + 2, entry);
        entry = page_entry(t + 3);
        request(true, buf);
        deposit(false, buf ^ 1);
        deposit(true, buf);
      }
    }
  };
  if (r0 + wave * 32 < rows) walk(std::true_type{}); else walk(std::false_type{});
  if (t_first < t_last) {
    volatile int* flag = (volatile int*)smem;   // the tiles are used up
    __syncthreads();
    if (threadIdx.x == 0) *flag = 0;
    __syncthreads();
    if (w.not_finite() && lane == 0) *flag = 1;
    __syncthreads();
    const bool again = *flag != 0;
    __syncthreads();
    if (again) {                                // tile by tile
      w.start();
      for (int t = t_first; t < t_last; ++t) {
        rows_of(t, page_entry(t));
        __syncthreads();
        request(true, 0);
        request(false, 0);
        deposit(true, 0);
        deposit(false, 0);
        publish();
        w.template plain_tile<NB, true>(k_tile(0), v_tile(0), t * BN, [] {});
      }
    }
  }
  w.l = half_sum(w.l);
  w.store();
}

// The same 32 rows in every wave, 32 keys of its own at a time: wave k takes blocks k, k + NW, ... of the range.
template <typename T, bool FP8, bool CAP, int D>
__device__ __forceinline__ void fd_key_tile(const PrefillArgs& a, const PrefillItem& it, char* smem) {
  using W = PrefillWave<T, FP8, CAP, D>;
  using Tile = PrefillTile<D>;
  constexpr int NW = key_tile_waves(D), MB = W::MB;
  constexpr int kTileB = 32 * Tile::kRowB;
  constexpr int kLoads = 32 * W::kInChunks / 64;          // loads per lane and operand
  constexpr int kUnit = row_tile_keys(D);                 // ranges are whole row-tile keys, as planned
  constexpr int kState = D * 32 + 64;                     // floats of a wave's state: O, m, l
  static_assert(2 * NW * kTileB <= kPrefillLds && (NW - 1) * kState * 4 <= kPrefillLds, "[NW][K tile, V tile]; the states");
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = it.j * 32, rows = it.n_q * a.G;
  W w(a, it, r0);
  const int lane = w.lane;
  const int hi_all = max(it.limit_of(a, min(r0 + 31, rows - 1)), 0);
  const int all_tiles = (hi_all + kUnit - 1) / kUnit;
  const int per_split = max((all_tiles + it.splits - 1) / it.splits, it.min_tiles);
  const int lo = min(it.split * per_split, all_tiles) * kUnit;
  const int hi = min(hi_all, min((it.split + 1) * per_split, all_tiles) * kUnit);
  char* k_tile = smem + wave * 2 * kTileB;
  char* v_tile = k_tile + kTileB;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem + wave * 2 * kTileB;

  // ---- loads of a block: 16-byte chunk n = 64 i + lane.  fp8: into registers, `f8`
  auto page_entry = [&](int t0) { return it.page_entry(a, t0 + (lane & 31)); };
  using Raw = u32x4[FP8 ? 2 * kLoads : 1];
  auto request = [&](bool is_k, int row, Raw& f8) {
    if (!FP8) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // what was read of the block before has arrived
#pragma unroll (kLoads > 8 ? 4 : kLoads)
    for (int i = 0; i < kLoads; ++i) {
      const int n = i * 64 + lane;
      const int r = n / W::kInChunks, ch = n % W::kInChunks;
      const char* src = (is_k ? w.kb : w.vb) + (uint64_t)(uint32_t)__shfl(row, r) * (is_k ? w.sk_b : w.sv_b)
                        + (W::source_chunk(is_k, r, ch) << 4);
      if constexpr (FP8)
        f8[is_k ? i : kLoads + i] = load_stream_b128(src);
      else
        load_to_lds_b128<true>(src, __builtin_amdgcn_readfirstlane(lds0 + (is_k ? 0 : kTileB) + i * 1024));
    }
  };
  auto deposit = [&](Raw& f8) {
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) {
      const int n = i % kLoads * 64 + lane;
      W::deposit(i < kLoads, i < kLoads ? k_tile : v_tile, n / W::kInChunks, n % W::kInChunks, f8[i]);
    }
    wave_lds_fence();
  };
  // No barrier.  16-bit caches: one block deep per wave, K of the next block is requested when this one's scores are done, V
  // when its product is; the waves of two workgroups cover each other's waits.  fp8: kDeep blocks in registers, a block is
  // requested as soon as the one kDeep before it is in LDS (own keys of 128 sequences: two deep is level with one and needs
  // more registers).  Page entries are read a block ahead and before that block's requests: loads return in order, and the
  // wait for an entry is one for what came before it.
  auto walk = [&](auto careful_tag) {
    constexpr bool CAREFUL = decltype(careful_tag)::value;
    constexpr int kStep = 32 * NW;
    w.start();
    int t0 = lo + 32 * wave;
    if (wave >= NW || t0 >= hi) return;
    int entry = page_entry(t0), ahead = page_entry(t0 + kStep);
    auto next_row = [&](int t) {                // the lane's row of block t (past the end: the last key's)
      const int row = it.pool_row(a, t + (lane & 31), entry);
      entry = ahead;
      ahead = page_entry(t + 2 * kStep);
      return row;
    };
    if constexpr (FP8) {
      constexpr int kDeep = 1;
      Raw raw[kDeep];
      auto request_both = [&](int t, Raw& f8) {
        const int row = next_row(t);
        request(true, row, f8);
        request(false, row, f8);
      };
#pragma unroll
      for (int d = 0; d < kDeep; ++d) request_both(t0 + d * kStep, raw[d]);
      for (; t0 < hi; t0 += kDeep * kStep) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {       // (as a plain loop head dim 256 spills 64 - 120 registers, in this form 17:
          const int t = t0 + d * kStep;         // 161 -> 92 us a step of eight sequences of 8000 tokens)
          if (t >= hi) break;
          deposit(raw[d]);
          request_both(t + kDeep * kStep, raw[d]);
          w.template plain_tile<1, CAREFUL>(k_tile, v_tile, t, [] {});
        }
      }
    } else {
      Raw none;
      int row = next_row(t0);
      request(true, row, none);
      request(false, row, none);
      for (; t0 < hi; t0 += kStep) {
        const int next = t0 + kStep;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        w.template plain_tile<1, CAREFUL>(k_tile, v_tile, t0, [&] {
          if (next < hi) {
            row = next_row(next);
            request(true, row, none);
          }
        });
        if (next < hi) request(false, row, none);
      }
    }
  };
  walk(std::false_type{});
  if (w.not_finite()) walk(std::true_type{});
  w.l = half_sum(w.l);
  // ---- join the states of the waves that had keys in wave 0
  float* st = (float*)smem;
  __syncthreads();
  if (wave > 0 && wave < NW && lo + 32 * wave < hi) {
    float* mine = st + (wave - 1) * kState;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(f32x4*)(mine + ((mb * 4 + i) * 64 + lane) * 4) = f32x4{w.o[mb][4 * i], w.o[mb][4 * i + 1], w.o[mb][4 * i + 2], w.o[mb][4 * i + 3]};
    if (w.half == 0) {
      mine[D * 32 + w.l32] = w.m;
      mine[D * 32 + 32 + w.l32] = w.l;
    }
  }
  __syncthreads();
  if (wave > 0) return;
  const int others = min(NW, (hi - lo + 31) / 32) - 1;   // waves 1 .. others had keys
  float top = w.m;
  for (int k = 0; k < others; ++k) top = fmaxf(top, st[k * kState + D * 32 + w.l32]);
  const float own = fd_exp2(w.m - top);
  w.m = top;
  w.l *= own;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) w.o[mb] *= own;
  for (int k = 0; k < others; ++k) {
    const float* his = st + k * kState;
    const float f = fd_exp2(his[D * 32 + w.l32] - top);
    w.l += f * his[D * 32 + 32 + w.l32];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = *(const f32x4*)(his + ((mb * 4 + i) * 64 + lane) * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) w.o[mb][4 * i + e] += f * x[e];
      }
  }
  w.store();
}

// T: query and product type.  FP8: e4m3 cache.  CAP: soft-capped scores.  D: head dim.  ROWS: tiles of 128 rows, else of 32.
// The bodies keep two workgroups of four waves on a CU, one with a head dim of 256: at most 256 registers a lane, 512 there.
// What does not fit goes to scratch.  Registers spilled (bytes a lane), without and with a soft cap: none with a head dim of
// 64; key tiles none with 128, 9 and 18 (40, 72) with 256, over fp8 17 and 0 (72, 0); row tiles, whose kernel holds both
// bodies, 6 and 8 (28, 36) with 128, over fp8 4 and 8 (20, 36), and 25 and 37 (76, 104) with 256, over fp8 43 and 32 (136, 124).
template <typename T, bool FP8, bool CAP, int D, bool ROWS>
__global__ void __launch_bounds__(64 * kPrefillWaves, D == 256 ? 1 : 2) fd_prefill_kernel(const PrefillArgs a) {
  extern __shared__ __align__(1024) char smem[];
  PrefillItem it;
  bool own;
  if (!fd_find_item(a, ROWS ? 32 * kPrefillWaves : 32, it, own)) return;
  if constexpr (ROWS) {
    if (!own) {
      fd_row_tile<T, FP8, CAP, D>(a, it, smem);
      return;
    }
  }
  fd_key_tile<T, FP8, CAP, D>(a, it, smem);
}

template <typename T, bool FP8, int D>
int launch_prefill(hipStream_t stream, const PrefillArgs& args, bool row_tiles) {
  PrefillArgs a = args;
  const int bm = row_tiles ? 32 * kPrefillWaves : 32;
  const int64_t tiles = ((int64_t)a.total_q * a.G + (int64_t)a.batch * (bm - 1)) / bm;   // sum of ceil(rows_b / bm) at most
  const int64_t own = a.own_splits > 0 ? (int64_t)a.total_q * ((a.G + 31) / 32) * a.own_splits : 0;
  const int64_t wgs = (tiles * a.splits + own) * a.Hkv;
  if (wgs >= ((int64_t)1 << 31)) return FD_ERR_TOO_LARGE;
  if (wgs == 0) return FD_OK;
  a.group_units = (int32_t)(tiles * a.splits);
  a.own_units = (int32_t)own;
  const bool cap = a.soft_cap > 0.f;
  auto kern = row_tiles ? (cap ? fd_prefill_kernel<T, FP8, true, D, true> : fd_prefill_kernel<T, FP8, false, D, true>)
                        : (cap ? fd_prefill_kernel<T, FP8, true, D, false> : fd_prefill_kernel<T, FP8, false, D, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(64 * kPrefillWaves), kPrefillLds, stream, a);
  return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH;
}

}  // namespace
