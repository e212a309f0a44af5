// Attention of many query rows over packed keys or over the paged cache (gfx950): prompts, chunks of prompts, drafted
// tokens, and the prefix part of a shared-prefix decode step.
//
// out[i,h] = sum_j softmax_j(scale q[i,h].k[j,h/G]) v[j,h/G] over the keys j that row i sees: j < n_k, and in the causal
// form j <= i + n_k - n_q (the last query sees the last key).  One pass over the keys with the running maximum m and sum
// l of the softmax; the accumulator is rescaled only when the maximum has grown by more than 2^8 (as in
// fd_softmax_step).
//
// Rows: the G query heads of a KV head share its keys, so a row is a (token, head of the group) pair, r = token * G + head,
// and a workgroup owns 32 * WR consecutive rows of one sequence and one KV head: a causal tile of G = 4 spans a quarter
// of the tokens that 32 * WR rows of one head would, and wastes that much less on its diagonal.
// Both products run on v_mfma_f32_32x32x16 with the scores transposed, S^T[token][row] = K Q^T and
// O^T[dim][row] += V^T P^T: lane l then holds scores of row l % 32 only -- 16 of the 32 tokens of a block, tokens
// 8 (i / 4) + 4 (l / 32) + i % 4 -- so a row's maximum and sum are in-lane reductions plus one exchange between the wave
// halves, and those tokens are, eight at a time, exactly the k indices that the lane supplies as B operand of the second
// product: P never leaves its registers.  V comes from LDS through the transposing read (ds_read_b64_tr_b16): 16 lanes
// read four tokens of 16 dims and receive four tokens of one dim each.
// Keys go global -> LDS without passing through registers (16-bit caches; 16 bytes a lane), two tiles deep.  The LDS image
// of such a load is lane-linear, so rows are swizzled at the source: lane c of a row fetches the 16-byte chunk c ^ f(row),
// with f chosen so that the 128-bit K reads (32 rows of one chunk column) and the transposing V reads (8 rows of 64 bytes)
// both touch all 64 banks.  An fp8 cache is converted once per workgroup on its way to LDS (exact) instead.
//
// Tokens past a sequence's length are never fetched: the row address is clamped to the last token, and what such a row
// holds is masked.  A masked score has weight 0, and 0 times a V row that is finite is 0; a V row that holds an infinity
// or NaN would turn rows that do not see it into NaN, so a workgroup whose result is not finite runs once more with the
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
__device__ __forceinline__ void load_to_lds_b128(const void* src, uint32_t lds_base) {
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

// T: query and product type.  FP8: e4m3 cache.  CAP: soft-capped scores.  D: head dim.  WR row groups x WT token groups of waves, BN tokens a tile.
template <typename T, bool FP8, bool CAP, int D, int WR, int WT, int BN>
__global__ void __launch_bounds__(64 * WR * WT, D == 256 ? 1 : 2) fd_prefill_kernel(const PrefillArgs a) {
  using Tile = PrefillTile<D>;
  constexpr int NW = WR * WT;
  constexpr int BM = 32 * WR;
  constexpr int NT = BN / WT;              // tokens of a tile that a wave works on
  constexpr int NB = NT / 32;              // ... in blocks of 32
  constexpr int KS = D / 16;               // k steps of the scores
  constexpr int MB = D / 32;               // dim blocks of the output
  constexpr int kTileB = BN * Tile::kRowB; // bytes of a K (or V) tile in LDS
  static_assert(NT % 32 == 0 && BN * Tile::kChunks % (64 * NW) == 0, "tile shape");
  static_assert(4 * kTileB <= 65536, "two tiles of K and V within the reach of the direct loads' 16-bit LDS offset");
  extern __shared__ __align__(1024) char smem[];             // [2][K tile, V tile]

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave % WR, wt = wave / WR;
  const int half = lane >> 5, l32 = lane & 31;

  // ---- work item: KV head fastest (the eight XCDs take neighbouring workgroups in turn, so with eight KV heads each
  // XCD's L2 holds one head's keys), then the key range, then the row tile
  const int kvh = blockIdx.x % a.Hkv;
  int unit = blockIdx.x / a.Hkv, slot, split, splits, min_tiles;     // slot: of the partial
  int b = -1, q_start = 0, n_q = 0, k_start = 0, n_k = 0, j = 0;
  const int32_t* table = a.bt;
  if (a.own_splits > 0 && unit >= a.group_units) {
    // a sequence's own keys behind its group's prefix
    unit -= a.group_units;
    splits = a.own_splits;
    min_tiles = a.own_min_tiles;
    split = unit % splits;
    slot = a.splits + split;
    const int rest = unit / splits, tiles = (a.G + BM - 1) / BM;
    q_start = rest / tiles;
    j = rest - q_start * tiles;
    if (q_start >= a.total_q) return;
    n_q = 1;
    n_k = min(max(a.own_lens[q_start], 0), a.own_max_pages * a.P);
    table = a.own_bt + (int64_t)q_start * a.own_sbt;
  } else {
    splits = a.splits;
    min_tiles = a.min_tiles;
    split = slot = unit % splits;
    const int tile = unit / splits;
    // The row tile of the list: sequences with the most keys first (in blocks of 64 sequences, one a lane), the tiles of a
    // sequence from its end, where a causal row sees the most -- short work fills in behind long.  In index order the last
    // long sequence of a batch runs alone at the end.
    for (int b0 = 0, base = 0; b0 < a.batch; b0 += 64) {
      const int mine = b0 + lane;
      int qs = 0, nq = 0, ks = 0, nk = -1, tiles = 0;
      if (mine < a.batch) {
        fd_prefill_span(a, mine, qs, nq);
        if (a.bt) {
          nk = min(max(a.kv_lens[mine], 0), a.max_pages * a.P);
        } else {
          ks = min(max(a.cu_k[mine], 0), a.total_k);
          nk = min(max(a.cu_k[mine + 1], ks), a.total_k) - ks;
        }
        tiles = (nq * a.G + BM - 1) / BM;
      }
      int before = 0, total = 0;                // tiles of the sequences that come before this lane's; of all
      const int n = min(64, a.batch - b0);
      for (int i = 0; i < n; ++i) {
        const int k_i = __builtin_amdgcn_readlane(nk, i), t_i = __builtin_amdgcn_readlane(tiles, i);
        before += k_i > nk || (k_i == nk && i < lane) ? t_i : 0;
        total += t_i;
      }
      const int at = tile - base - before;
      const uint64_t here = __ballot(at >= 0 && at < tiles);
      if (here) {
        const int w = __builtin_ctzll(here);
        b = b0 + w;
        q_start = __builtin_amdgcn_readlane(qs, w);
        n_q = __builtin_amdgcn_readlane(nq, w);
        k_start = __builtin_amdgcn_readlane(ks, w);
        n_k = __builtin_amdgcn_readlane(nk, w);
        j = __builtin_amdgcn_readlane(tiles, w) - 1 - __builtin_amdgcn_readlane(at, w);
        break;
      }
      base += total;
    }
    if (b < 0) return;
    if (table) table += (int64_t)b * a.sbt;
  }

  const int rows = n_q * a.G;
  // keys that row r of the sequence sees: [0, limit)
  auto token_of = [&](int r) { return (int)(((uint64_t)(uint32_t)r * a.g_magic) >> a.g_shift); };
  auto limit_of = [&](int r) { return a.causal ? min(n_k, token_of(r) + 1 + n_k - n_q) : n_k; };
  const int r0 = j * BM;
  const int row = min(r0 + wr * 32 + l32, rows - 1);   // rows past the end repeat the last one and are not stored
  const bool real_row = r0 + wr * 32 + l32 < rows;
  const int q_tok = token_of(row), q_head = row - q_tok * a.G;
  const int my_limit = limit_of(row);
  const int wave_lo = limit_of(min(r0 + wr * 32, rows - 1));            // the wave's rows see at least this many keys
  const int wg_hi = limit_of(min(r0 + BM - 1, rows - 1));
  const int all_tiles = (max(wg_hi, 0) + BN - 1) / BN;
  const int per_split = max((all_tiles + splits - 1) / splits, min_tiles);
  const int t_first = min(split * per_split, all_tiles);
  const int t_last = min(t_first + per_split, all_tiles);

  // ---- Q^T as B operand: lane (row, half) holds dims 16 ks + 8 half .. + 7
  u32x4 qf[KS];
  {
    const char* qp = (const char*)a.q + 2 * ((int64_t)(q_start + q_tok) * a.sq_t + (int64_t)(kvh * a.G + q_head) * a.sq_h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *(const u32x4*)(qp + 32 * ks + 16 * half);
  }
  float c = a.sm_scale;
  if (FP8) c *= a.k_scale[kvh];
  float cap = 0.f, cap_in = 0.f;
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

  // ---- addresses
  const int ksw = Tile::k_swz(l32);                     // row of a K read: l32 + a multiple of 32
  const int k_lane = (wt * NT + l32) * Tile::kRowB + ((half ^ ksw) << 4);
  const int vi = lane & 15;
  const int v_tok = wt * NT + 4 * half + (vi >> 2);
  const int v_lane = v_tok * Tile::kRowB + ((lane >> 4) & 1) * 32 + (vi & 3) * 8;
  const int v_swz = Tile::v_swz(v_tok) << 4;            // the same for all token steps of 8
  const char* kb = (const char*)a.k + (FP8 ? 1 : 2) * ((int64_t)kvh * a.sk_h);
  const char* vb = (const char*)a.v + (FP8 ? 1 : 2) * ((int64_t)kvh * a.sv_h);
  const uint32_t sk_b = (uint32_t)a.sk_t * (FP8 ? 1 : 2), sv_b = (uint32_t)a.sv_t * (FP8 ? 1 : 2);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;

  // The token row in the pool of token t0 + lane of a tile (lanes past BN repeat the last): page entry first, so that it
  // can be requested a tile early.
  auto page_entry = [&](int t) -> int {
    if (!table) return 0;
    const int tok = min(t * BN + min(lane, BN - 1), n_k - 1);
    const int pg = (int)(((uint64_t)(uint32_t)tok * a.p_magic) >> a.p_shift);
    return table[pg];
  };
  auto pool_row = [&](int t, int entry) -> int {
    const int tok = min(t * BN + min(lane, BN - 1), n_k - 1);
    if (!table) return k_start + tok;
    const int pg = (int)(((uint64_t)(uint32_t)tok * a.p_magic) >> a.p_shift);
    return min(max(entry, 0), a.num_pages - 1) * a.P + (tok - pg * a.P);
  };

  // ---- tile loads.  16-bit: chunk n = (i NW + wave) 64 + lane of the tile's LDS image.  fp8: through registers.
  constexpr int kChunksLoaded = FP8 ? D / 16 : Tile::kChunks;         // 16-byte chunks of a row in memory
  constexpr int kLoads = BN * kChunksLoaded / (64 * NW);              // loads per lane and operand
  int pr[kLoads];                                                     // pool rows that this lane fetches from
  u32x4 f8k[FP8 ? kLoads : 1], f8v[FP8 ? kLoads : 1];
  auto rows_of = [&](int rows_of_tile) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) pr[i] = __shfl(rows_of_tile, ((i * NW + wave) * 64 + lane) / kChunksLoaded);
  };
  // (a pool has fewer than 2^31 rows and a row stride fits 32 bits: one 32 x 32 -> 64 bit multiply)
  auto request = [&](bool is_k, int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int n = (i * NW + wave) * 64 + lane;
      const int r = n / kChunksLoaded, ch = n % kChunksLoaded;
      const char* src = (is_k ? kb : vb) + (uint64_t)(uint32_t)pr[i] * (is_k ? sk_b : sv_b);
      if constexpr (FP8) {
        (is_k ? f8k : f8v)[i] = *(const u32x4*)(src + (ch << 4));
      } else {
        const uint32_t dst = lds0 + (2 * buf + (is_k ? 0 : 1)) * kTileB + (i * NW + wave) * 1024;
        load_to_lds_b128(src + ((ch ^ (is_k ? Tile::k_swz(r) : Tile::v_swz(r))) << 4), __builtin_amdgcn_readfirstlane(dst));
      }
    }
  };
  auto deposit = [&](bool is_k, int buf) {   // fp8: convert what `request` fetched and put it into LDS
    if constexpr (FP8) {
      char* at = smem + (2 * buf + (is_k ? 0 : 1)) * kTileB;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int n = (i * NW + wave) * 64 + lane;
        const int r = n / kChunksLoaded, ch = n % kChunksLoaded;
        const u32x4 raw = (is_k ? f8k : f8v)[i];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 x = {Mma<T>::from_fp8(raw[2 * h], false), Mma<T>::from_fp8(raw[2 * h], true),
                           Mma<T>::from_fp8(raw[2 * h + 1], false), Mma<T>::from_fp8(raw[2 * h + 1], true)};
          *(u32x4*)(at + r * Tile::kRowB + (((2 * ch + h) ^ (is_k ? Tile::k_swz(r) : Tile::v_swz(r))) << 4)) = x;
        }
      }
    }
  };
  auto publish = [&] {   // what was requested is in LDS, for every wave, and nobody reads what is requested next
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  // ---- the pieces of a tile's work
  auto k_frag = [&](int buf, int ks, int tb) {
    return lds_read_b128(smem + 2 * buf * kTileB + (k_lane ^ (ks << 5)) + tb * 32 * Tile::kRowB);
  };
  auto v_frag = [&](int buf, int st, int mb) -> u32x4 {
    const char* vp = smem + (2 * buf + 1) * kTileB + v_lane + st * 16 * Tile::kRowB + ((mb << 6) ^ v_swz);
    const u32x2 lo = lds_read_tr(vp), hi = lds_read_tr(vp + 8 * Tile::kRowB);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  // soft cap and mask of tile t's raw scores (a wave-uniform branch, which most tiles pass by)
  auto finish_scores = [&](int t, f32x16 (&s)[NB]) {
    if constexpr (CAP) {
#pragma unroll
      for (int tb = 0; tb < NB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = fd_exp2(s[tb][i] * cap_in);
          s[tb][i] = __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + e), cap);   // tanh(y) = 1 - 2 / (1 + e^2y)
        }
    }
    const int t0 = t * BN + wt * NT;       // first token of this wave's part
    if (t0 + NT > wave_lo) {
      const int see = my_limit - t0 - 4 * half;
#pragma unroll
      for (int tb = 0; tb < NB; ++tb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[tb][i] = tb * 32 + 8 * (i / 4) + i % 4 < see ? s[tb][i] : -INFINITY;
    }
  };

  f32x16 o[MB];
  float m, l;
  auto start = [&] {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) o[mb] = f32x16{};
    m = -3.0e38f;     // below every score: a row that sees nothing keeps l = 0
    l = 0.f;
  };
  // the reference point follows the maximum `mx` of the next tile's raw scores (this lane's tokens of its row)
  auto move_reference = [&](float mx) {
    const float top = fmaxf(m, half_max(mx) * c);
    const float m_new = top - m > 8.0f ? top : m;
    if (__any(m_new > m)) {
      const float alpha = fd_exp2(m - m_new);
      l *= alpha;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[mb] *= alpha;
      m = m_new;
    }
  };

  // One tile of the pipelined walk.  On entry `cur` holds tile t's finished scores, `mx` their maximum over this lane, pr
  // the pool rows of tile t + 1, whose K is on its way, like V of tile t.  The scores of tile t + 1 are computed while the
  // weights of tile t are (one MFMA and a few weights at a time: the matrix pipe works on one while the vector pipe does
  // the others), and their maximum while V of tile t is multiplied.
  constexpr int E = 16 * NB;               // scores of a lane
  auto step = [&](int t, int& entry, float& mx, f32x16 (&cur)[NB], f32x16 (&nxt)[NB], auto next_tag) {
    constexpr bool NEXT = decltype(next_tag)::value;
    const int buf = (t - t_first) & 1;
    publish();
    const bool more = NEXT && t + 2 < t_last;
    if constexpr (NEXT) {
      request(false, buf ^ 1);             // V of t + 1 over V of t - 1
      if (more) {
        rows_of(pool_row(t + 2, entry));
        entry = page_entry(t + 3);
        request(true, buf);                // K of t + 2 over K of t
      }
    }
    move_reference(mx);
    // P is rounded to the query's type for the second product (the sum l is not): half a step, 2^-8 (bf16) or 2^-11 (fp16)
    // of each weight, of both signs -- less in their sum than the rounding of the output itself
    u32x4 pf[NT / 16];
    float sum0 = 0.f, sum1 = 0.f;
    auto weights = [&](int e0, int e1) {   // scores e0 .. e1 - 1, in pairs
#pragma unroll
      for (int e = e0; e < e1; e += 2) {
        const float p0 = fd_exp2(__builtin_fmaf(cur[e / 16][e % 16], c, -m));
        const float p1 = fd_exp2(__builtin_fmaf(cur[e / 16][e % 16 + 1], c, -m));
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
        for (int tb = 0; tb < NB; ++tb) nxt[tb] = Mma32<T>::run(k_frag(buf ^ 1, ks, tb), qf[ks], nxt[tb]);
        weights(E * ks / KS & ~1, E * (ks + 1) / KS & ~1);
      }
      // pinned here: left to itself the compiler moves the weights behind the branches of finish_scores, next to their use
#pragma unroll
      for (int st = 0; st < NT / 16; ++st) asm volatile("" : "+v"(pf[st]));
      l += sum0 + sum1;
      asm volatile("" : "+v"(l));
      finish_scores(t + 1, nxt);
    } else {
      weights(0, E);
      l += sum0 + sum1;
    }
    mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < NT / 16; ++st)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        o[mb] = Mma32<T>::run(v_frag(buf, st, mb), pf[st], o[mb]);
        if constexpr (NEXT) {
          constexpr int N = NT / 16 * MB;  // MFMAs of this product
          const int at = st * MB + mb;
#pragma unroll
          for (int e = E * at / N; e < E * (at + 1) / N; ++e) mx = fmaxf(mx, nxt[e / 16][e % 16]);
        }
      }
    if constexpr (FP8 && NEXT) {
      deposit(false, buf ^ 1);
      if (more) deposit(true, buf);
    }
  };

  auto walk = [&] {
    start();
    if (t_first >= t_last) return;
    rows_of(pool_row(t_first, page_entry(t_first)));
    int entry = page_entry(t_first + 1);
    request(true, 0);
    request(false, 0);
    if constexpr (FP8) {
      deposit(true, 0);
      deposit(false, 0);
    }
    publish();
    if (t_first + 1 < t_last) {
      rows_of(pool_row(t_first + 1, entry));
      entry = page_entry(t_first + 2);
      request(true, 1);
    }
    f32x16 s0[NB], s1[NB];
#pragma unroll
    for (int tb = 0; tb < NB; ++tb) s0[tb] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) s0[tb] = Mma32<T>::run(k_frag(0, ks, tb), qf[ks], s0[tb]);
    finish_scores(t_first, s0);
    float mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) mx = fmaxf(mx, s0[e / 16][e % 16]);
    if constexpr (FP8) {
      if (t_first + 1 < t_last) deposit(true, 1);
    }
    int t = t_first;
    for (; t + 2 < t_last; t += 2) {       // two tiles a turn: the two sets of scores change places without copies
      step(t, entry, mx, s0, s1, std::true_type{});
      step(t + 1, entry, mx, s1, s0, std::true_type{});
    }
    if (t + 1 < t_last) {
      step(t, entry, mx, s0, s1, std::true_type{});
      step(t + 1, entry, mx, s1, s0, std::false_type{});
    } else {
      step(t, entry, mx, s0, s1, std::false_type{});
    }
  };

  // A wave whose rows are all past the end only fetches.
  auto walk_idle = [&] {
    start();
    if (t_first >= t_last) return;
    rows_of(pool_row(t_first, page_entry(t_first)));
    int entry = page_entry(t_first + 1);
    request(true, 0);
    request(false, 0);
    deposit(true, 0);
    deposit(false, 0);
    publish();
    if (t_first + 1 < t_last) {
      rows_of(pool_row(t_first + 1, entry));
      entry = page_entry(t_first + 2);
      request(true, 1);
      deposit(true, 1);
    }
    for (int t = t_first; t < t_last; ++t) {
      const int buf = (t - t_first) & 1;
      publish();
      if (t + 1 >= t_last) continue;
      request(false, buf ^ 1);
      if (t + 2 < t_last) {
        rows_of(pool_row(t + 2, entry));
        entry = page_entry(t + 3);
        request(true, buf);
      }
      deposit(false, buf ^ 1);
      if (t + 2 < t_last) deposit(true, buf);
    }
  };

  // The second walk of a workgroup whose result was not finite: tile by tile, no pipeline.
  auto walk_careful = [&] {
    start();
    for (int t = t_first; t < t_last; ++t) {
      rows_of(pool_row(t, page_entry(t)));
      __syncthreads();
      request(true, 0);
      request(false, 0);
      deposit(true, 0);
      deposit(false, 0);
      publish();
      f32x16 s[NB];
#pragma unroll
      for (int tb = 0; tb < NB; ++tb) s[tb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int tb = 0; tb < NB; ++tb) s[tb] = Mma32<T>::run(k_frag(0, ks, tb), qf[ks], s[tb]);
      finish_scores(t, s);
      const int t0 = t * BN + wt * NT;
      const bool masked = t0 + NT > wave_lo;
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) mx = fmaxf(mx, s[e / 16][e % 16]);
      move_reference(mx);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        s[e / 16][e % 16] = fd_exp2(__builtin_fmaf(s[e / 16][e % 16], c, -m));
        l += s[e / 16][e % 16];
      }
#pragma unroll
      for (int st = 0; st < NT / 16; ++st) {
        u32x4 pf;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          pf[w] = Mma<T>::pack(s[st / 2][8 * (st % 2) + 2 * w], s[st / 2][8 * (st % 2) + 2 * w + 1]);
#pragma unroll 1
        for (int mb = 0; mb < MB; ++mb) {
          u32x4 vf = v_frag(0, st, mb);
          if (masked) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t e = vf[w] & Mma32<T>::kExp;
              if ((e & 0xffffu) == (Mma32<T>::kExp & 0xffffu)) vf[w] &= 0xffff0000u;
              if ((e >> 16) == (Mma32<T>::kExp >> 16)) vf[w] &= 0xffffu;
            }
          }
#pragma unroll
          for (int k = 0; k < MB; ++k)     // (registers have no run-time index)
            if (k == mb) o[k] = Mma32<T>::run(vf, pf, o[k]);
        }
      }
      if (!masked) continue;
      // the non-finite V values of this tile, for the rows that see them: lane (row, half) owns dims 32 mb + 8 i + 4 half
      // .. + 3
      for (int n = 0; n < NT; ++n) {
        if (t0 + n >= my_limit) continue;
        const int r = wt * NT + n;
        const char* vr = smem + kTileB + r * Tile::kRowB;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d0 = 32 * mb + 8 * i + 4 * half;
            const u32x2 w = *(const u32x2*)(vr + ((((d0 >> 3) ^ Tile::v_swz(r)) << 4) | ((d0 & 4) << 1)));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint16_t bits = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
              if ((bits & (uint16_t)Mma32<T>::kExp) == (uint16_t)Mma32<T>::kExp)
                o[mb][4 * i + e] += (float)__builtin_bit_cast(T, bits);
            }
          }
      }
    }
  };
  if (r0 + wr * 32 < rows) walk(); else walk_idle();
  if (t_first < t_last) {
    // any value that is not finite?  (x - x is 0 for finite x)
    float probe = l - l;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) probe += o[mb][i] - o[mb][i];
    volatile int* flag = (volatile int*)smem;   // the tiles are used up
    __syncthreads();
    if (threadIdx.x == 0) *flag = 0;
    __syncthreads();
    if (__any(!(probe == 0.f)) && lane == 0) *flag = 1;
    __syncthreads();
    const bool again = *flag != 0;
    __syncthreads();
    if (again) walk_careful();
  }

  // ---- join the token groups, store
  l = half_sum(l);
  if constexpr (WT > 1) {
    static_assert(WT == 2, "two token groups");
    static_assert(WR * (D * 32 + 64) * 4 <= 4 * kTileB, "the second group's state fits over the tiles");
    float* st = (float*)smem + wr * (D * 32 + 64);
    __syncthreads();
    if (wt == 1) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[(mb * 16 + i) * 64 + lane] = o[mb][i];
      if (half == 0) {
        st[D * 32 + l32] = m;
        st[D * 32 + 32 + l32] = l;
      }
    }
    __syncthreads();
    if (wt == 1) return;
    const float m1 = st[D * 32 + l32], l1 = st[D * 32 + 32 + l32];
    const float top = fmaxf(m, m1);
    const float f0 = fd_exp2(m - top), f1 = fd_exp2(m1 - top);
    l = l * f0 + l1 * f1;
    m = top;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[mb][i] = o[mb][i] * f0 + st[(mb * 16 + i) * 64 + lane] * f1;
  }
  if (!real_row) return;
  float inv = l != 0.f ? 1.0f / l : 0.f;
  const float lse = l != 0.f ? m * FD_LN2 + __logf(l) : -INFINITY;
  if (FP8) inv *= a.v_scale[kvh];
  const int64_t tok = q_start + q_tok;
  const int head = kvh * a.G + q_head;
  if (a.part) {
    const int64_t at = (tok * a.Hq + head) * (a.splits + a.own_splits) + slot;
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
        u32x2 w = {Mma<T>::pack(o[mb][4 * i] * inv, o[mb][4 * i + 1] * inv),
                   Mma<T>::pack(o[mb][4 * i + 2] * inv, o[mb][4 * i + 3] * inv)};
        *(u32x2*)(dst + 2 * (32 * mb + 8 * i + 4 * half)) = w;
      }
  }
}

template <typename T, bool FP8, int D, int WR, int WT, int BN>
int launch_prefill(hipStream_t stream, const PrefillArgs& args) {
  PrefillArgs a = args;
  constexpr int BM = 32 * WR;
  constexpr size_t lds = 4 * BN * 2 * D;
  const int64_t tiles = ((int64_t)a.total_q * a.G + (int64_t)a.batch * (BM - 1)) / BM;   // sum of ceil(rows_b / BM) at most
  const int64_t own = a.own_splits > 0 ? (int64_t)a.total_q * ((a.G + BM - 1) / BM) * a.own_splits : 0;
  const int64_t wgs = (tiles * a.splits + own) * a.Hkv;
  if (wgs >= ((int64_t)1 << 31)) return FD_ERR_TOO_LARGE;
  if (wgs == 0) return FD_OK;
  a.group_units = (int32_t)(tiles * a.splits);
  auto kern = a.soft_cap > 0.f ? fd_prefill_kernel<T, FP8, true, D, WR, WT, BN> : fd_prefill_kernel<T, FP8, false, D, WR, WT, BN>;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(64 * WR * WT), lds, stream, a);
  return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH;
}

}  // namespace
