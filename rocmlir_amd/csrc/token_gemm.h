// Products of token rows: an activation matrix whose rows belong to one group of weights or are spread over several
// (the experts of a mixture), the gradient of such weights, and the scales per token and channel of int8 operands.
//
// The tiles are those of gemm_conv_dlds.h and gemm_conv_kernel.h; what is added here is
//   * where a block's tile lies: the rows of group e are [offsets[e], offsets[e+1]), known on the device only, so the
//     grid covers the largest number of row tiles that M rows in G groups can make and every block finds its group
//     from the offsets by a scan over the lanes of a wave; blocks behind the last tile leave;
//   * the epilogue that multiplies int32 sums by channel_scale[n] and token_scale[m];
//   * the reduction over a group's rows (weight gradient), whose operands are addressed with 64-bit row positions.
// The reference has batched products with one size for all batch entries only (RockOps.td:63-99).
#pragma once
#include "gemm_conv_dlds.h"

namespace rk {

// ---- parameter blocks of a tile -----------------------------------------------------------
struct TokenTileParams : RockGemmParams {};
// results are f32, f16 or bf16
template <int OD> constexpr bool kTokenResult = OD == ROCK_F32 || OD == ROCK_F16 || OD == ROCK_BF16;
template <bool INT_ACC, typename F>
__device__ __forceinline__ void dispatch_tile_dtype(const TokenTileParams &p, F &&f) {
  switch (p.epi.out_dtype) {
  case ROCK_F32: f(std::integral_constant<int, ROCK_F32>{}); break;
  case ROCK_F16: f(std::integral_constant<int, ROCK_F16>{}); break;
  default: f(std::integral_constant<int, ROCK_BF16>{}); break;
  }
}

template <> struct AnyRowStart<TokenTileParams> : std::true_type {};

// ---- scales per token and channel -----------------------------------------------------
struct TokenScaleParams : TokenTileParams {
  const float *token_scale;   // of the tile's group: element m belongs to row m
  const float *channel_scale; // element n to column n; NULL: epi.scale
};
// (of its own: for a derived block the template over any parameter block would be the better match)
template <bool INT_ACC, typename F>
__device__ __forceinline__ void dispatch_tile_dtype(const TokenScaleParams &p, F &&f) {
  dispatch_tile_dtype<INT_ACC>(static_cast<const TokenTileParams &>(p), static_cast<F &&>(f));
}
__device__ __forceinline__ float token_scale_of(const TokenScaleParams &p, int m) {
  return p.token_scale && m < p.M ? p.token_scale[m] : 1.0f;
}
// One element: (sum - zero_point) * s[n] * t[m] + bias[n], clamped, every step one f32 operation, narrowed once
// afterwards.  A NaN stays one: it says that the row's activations held an infinity or a NaN.
__device__ __forceinline__ float scaled_value(int sum, float zero_point, float s, float t, float b, const RockEpilogue &e) {
  float v = ((float)sum - zero_point) * s * t;
  if (e.has_bias)
    v = v + b;
  if (e.activation && v == v)
    v = activation_fast(v, e);
  return v;
}
// four channels of row m, packed in the result's type
template <int OD>
__device__ __forceinline__ v4i token_convert4(const v4i &acc, const TokenScaleParams &p, int m, const void *bias, int n0) {
  static_assert(kTokenResult<OD>, "dispatch_tile_dtype must pick the list of these kernels");
  const RockEpilogue &e = p.epi;
  const float t = token_scale_of(p, m);
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) { // (channels behind the last one: any value, they are not stored)
    const int n = min(n0 + r, p.N - 1);
    v[r] = scaled_value(acc[r], (float)e.zero_point, p.channel_scale ? p.channel_scale[n] : e.scale, t,
                        e.has_bias ? ((const float *)bias)[n] : 0.0f, e);
  }
  return epilogue_pack4<OD>(v, e);
}
template <int OD>
__device__ __forceinline__ v4i token_convert4(const v4f &acc, const TokenTileParams &p, int, const void *bias, int n0) {
  return epilogue_convert4<false, OD>(acc, p.epi, bias, n0, p.N);
}

// Epilogue of the tiled kernels with these scales.  The raw sums go through the wave's LDS region, 32 rows at a time,
// and are scaled on the way out, where a lane holds eight consecutive columns of one row: its channel scales and biases
// are then the same for all its rows and are loaded once.  Scaled where they sit in the accumulators, every group of
// four would load its own, behind a bounds test each, once for every output type: four minutes of compilation and a
// hundred spilled scalar registers in the 256 x 256 tile (measured with seven types; it has three).
template <> struct HasRowScales<TokenScaleParams> : std::true_type {};
template <int DT, int MI, int NI, int NWAVES, int LDS_BYTES, typename Params>
__device__ __forceinline__ void row_scale_epilogue(typename MmaTraits<DT>::Acc (&acc)[MI][NI], const Params &p, int g,
                                                   void *Cptr, const void *aux, int m_wave, int n_wave, char *lds,
                                                   int wave, int lane) {
  constexpr int WTN = NI * 32, VEC = 8;
  constexpr int PITCH = WTN * 4 + 16, WBUF = 32 * PITCH;
  constexpr int LPR = WTN / VEC, RPI = 64 / LPR; // lanes per row, rows per pass
  static_assert(NWAVES * WBUF <= LDS_BYTES, "staging buffers must fit in the operand stages");
  const RockEpilogue &e = p.epi;
  const int lrow = lane & 31, lgrp = lane >> 5;
  char *wbuf = lds + wave * WBUF;
  const int rd_row = lane / LPR, rd_col = (lane % LPR) * VEC, n = n_wave + rd_col;
  float s[VEC], b[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) { // (columns behind the last one: any value, they are not stored)
    const int at = min(n + k, p.N - 1);
    s[k] = p.channel_scale ? p.channel_scale[at] : e.scale;
    b[k] = e.has_bias ? ((const float *)aux)[at] : 0.0f;
  }
  const float zero_point = (float)e.zero_point;
  __builtin_amdgcn_s_barrier(); // every wave is done reading the operand stages
  dispatch_tile_dtype<true>(p, [&](auto od_const) __attribute__((always_inline)) {
    constexpr int OD = decltype(od_const)::value, ES = OutElemSize<OD>::value;
    static_assert(kTokenResult<OD>, "dispatch_tile_dtype must pick the list of these kernels");
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *(v4i *)(wbuf + lrow * PITCH + (j * 32 + q * 8 + lgrp * 4) * 4) =
              v4i{acc[i][j][4 * q + 0], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      RK_WAVE_LDS_ORDER();
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += RPI) {
        const int row = r0 + rd_row, m = m_wave + i * 32 + row;
        const v4i lo = *(const v4i *)(wbuf + row * PITCH + rd_col * 4);
        const v4i hi = *(const v4i *)(wbuf + row * PITCH + rd_col * 4 + 16);
        const float t = token_scale_of(p, m);
        v4i out[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = scaled_value(h ? hi[k] : lo[k], zero_point, s[4 * h + k], t, b[4 * h + k], e);
          out[h] = epilogue_pack4<OD>(v, e);
        }
        if (m >= p.M)
          continue;
        char *dst = (char *)Cptr + ((int64_t)g * p.c_gs + (int64_t)m * p.c_ms + n) * ES;
        if constexpr (ES == 4) {
          store_row_piece<4>(dst, out[0], p.N - n);
          store_row_piece<4>(dst + 16, out[1], p.N - n - 4);
        } else {
          store_row_piece<2>(dst, v4i{out[0][0], out[0][1], out[1][0], out[1][1]}, p.N - n);
        }
      }
      RK_WAVE_LDS_ORDER();
    }
  });
}

// ---- which tile a block works on ---------------------------------------------------------
struct GroupTile {
  int e, row0, rows, tm, tn; // group, its first row and row count, tile inside the group
  int part, parts;           // which of how many parts of the tile
};

__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane * 4, v); }

// Boundaries are clamped to [0, M], and one that steps back is read as if it stood at the furthest one before it, so
// that whatever the offsets hold the groups are disjoint ranges of the M rows and every row tile is counted once.
struct GroupScan {
  int end, tiles; // running over the groups seen so far
};
// Lanes 0..63 take groups base..base+63: first row and row tiles before, up to and including the lane's group.
template <int BM>
__device__ __forceinline__ void scan_groups(const int32_t *offsets, int G, int M, int base, int lane, GroupScan &carry,
                                            int &start, int &end, int &tiles_end) {
  end = min(max(offsets[min(base + lane + 1, G)], 0), M); // (lanes behind the last group: its end, no tiles)
  start = lane_value(end, lane > 0 ? lane - 1 : 0);
  start = lane > 0 ? start : carry.end;
  if (__builtin_amdgcn_ballot_w64(end < start)) { // some boundary steps back: the running maximum
    end = max(end, carry.end);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int before = lane_value(end, lane >= d ? lane - d : lane);
      end = max(end, before);
    }
    start = lane_value(end, lane > 0 ? lane - 1 : 0);
    start = lane > 0 ? start : carry.end;
  }
  tiles_end = (end - start + BM - 1) / BM;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int before = lane_value(tiles_end, lane >= d ? lane - d : lane);
    tiles_end += lane >= d ? before : 0;
  }
  tiles_end += carry.tiles;
  carry.end = __builtin_amdgcn_readfirstlane(lane_value(end, 63));
  carry.tiles = __builtin_amdgcn_readfirstlane(lane_value(tiles_end, 63));
}

// The last tiles of a launch.  Tiles of 256 x 256 run one to a compute unit, so what is left after whole rounds over the
// chip would keep a few units busy for a full round while the others idle: up to half a round of such tiles is cut
// into halves (128 x 256), up to a quarter into quarters (128 x 128), which run side by side at the end.
constexpr int kUnits = 256;
__device__ __forceinline__ int tail_parts(int left) { return left * 4 <= kUnits ? 4 : left * 2 <= kUnits ? 2 : 1; }

// Tile number and part of this block among `total` tiles; false: the block has none.  Consecutive tiles go to one XCD
// (as decode_block does it) if `remap`.
template <bool SPLIT>
__device__ __forceinline__ bool block_tile(int total, bool remap, int &id, int &part, int &parts) {
  auto spread = [&](int i, int n) {
    const int per = n >> 3;
    return remap && i < (per << 3) ? (i & 7) * per + (i >> 3) : i;
  };
  id = blockIdx.x;
  part = 0;
  parts = 1;
  if constexpr (SPLIT) {
    const int full = total & ~(kUnits - 1), left = total - full;
    if (id >= full) {
      parts = tail_parts(left);
      if (id - full >= left * parts)
        return false;
      const int at = spread(id - full, left * parts);
      id = full + at / parts;
      part = at - at / parts * parts;
    } else {
      id = spread(id, full);
    }
    return true;
  }
  if (id >= total)
    return false;
  id = spread(id, total);
  return true;
}

// The tile of this block; false: the block has none.  Uniform over the block: every wave computes the same.
template <int BM, bool SPLIT = false>
__device__ __forceinline__ bool locate_tile(const int32_t *offsets, const RockGemmParams &p, GroupTile &t) {
  const int lane = threadIdx.x & 63;
  int start = 0, end = p.M, tiles_end = p.tiles_m, tile_rows = p.tiles_m;
  GroupScan first = {0, 0};
  if (offsets) {
    first.end = __builtin_amdgcn_readfirstlane(min(max(offsets[0], 0), p.M));
    GroupScan all = first;
    for (int base = 0; base < p.G; base += 64)
      scan_groups<BM>(offsets, p.G, p.M, base, lane, all, start, end, tiles_end);
    tile_rows = all.tiles;
  }
  int id;
  // (the tiles are at most the grid: the groups are disjoint)
  if (!block_tile<SPLIT>(tile_rows * p.tiles_n, p.xcd_remap != 0, id, t.part, t.parts))
    return false;
  t.e = 0;
  t.row0 = 0;
  t.rows = p.M;
  int tiles_m = p.tiles_m, in_group = id;
  if (offsets) {
    const int tile_row = id / p.tiles_n; // the group is found by it: a group's tiles are whole rows of tiles
    int base = 0;
    if (p.G > 64) {
      GroupScan seen = first;
      for (;; base += 64) { // (ends: tile_row < all.tiles, which the last pass reaches)
        scan_groups<BM>(offsets, p.G, p.M, base, lane, seen, start, end, tiles_end);
        if (tile_row < seen.tiles || base + 64 >= p.G)
          break;
      }
    }
    const uint64_t beyond = __builtin_amdgcn_ballot_w64(tiles_end > tile_row);
    const int at = beyond ? __builtin_ctzll(beyond) : 63;
    t.e = base + at;
    t.row0 = __builtin_amdgcn_readfirstlane(lane_value(start, at));
    t.rows = __builtin_amdgcn_readfirstlane(lane_value(end, at)) - t.row0;
    tiles_m = (t.rows + BM - 1) / BM;
    in_group -= (__builtin_amdgcn_readfirstlane(lane_value(tiles_end, at)) - tiles_m) * p.tiles_n;
  }
  // inside the group: blocks of group_m tile rows, walked down the columns, so that neighbours share operand tiles
  const int group_sz = p.group_m * p.tiles_n;
  const int grp = in_group / group_sz;
  const int first_m = grp * p.group_m;
  const int rows_here = min(tiles_m - first_m, p.group_m);
  const int in_grp = in_group - grp * group_sz;
  t.tm = first_m + in_grp % rows_here;
  t.tn = in_grp / rows_here;
  return true;
}

__device__ __forceinline__ int token_out_size(int od) { return od == ROCK_F32 ? 4 : 2; }

// Moves the operands to the tile's group and calls f(A, B, C, bias, params).
template <int DT, typename F>
__device__ __forceinline__ void with_group(const void *A, const void *B, void *C, const void *bias,
                                           const float *token_scale, const float *channel_scale,
                                           const RockTokenGemmParams &tp, const GroupTile &t, F &&f) {
  constexpr int ES = MmaTraits<DT>::ES;
  const RockGemmParams &p = tp.gemm;
  const void *a = (const char *)A + (int64_t)t.row0 * p.a_ms * ES;
  const void *b = (const char *)B + (int64_t)t.e * p.b_gs * ES;
  void *c = (char *)C + (int64_t)t.row0 * p.c_ms * token_out_size(p.epi.out_dtype);
  if constexpr (MmaTraits<DT>::INT_ACC) {
    TokenScaleParams q;
    static_cast<RockGemmParams &>(q) = p;
    q.M = t.rows;
    q.token_scale = token_scale ? token_scale + t.row0 : nullptr;
    q.channel_scale = channel_scale ? channel_scale + (int64_t)t.e * p.N : nullptr;
    f(a, b, c, bias, q);
  } else {
    TokenTileParams q;
    static_cast<RockGemmParams &>(q) = p;
    q.M = t.rows;
    f(a, b, c, bias, q);
  }
}

// One tile, or the block's part of it, in LDS that all of them share.
// Measured on MI355X.  256 x 256: bound by the matrix cores and their clock under load, 16384 bf16 rows over 8 groups of
// 2048 -> 4096 in 241 us (1.14 PFLOP/s; one dense product of that size 231), the gradient of the rows 252; int8 4096^3 with
// both scales 63 us (2.2 POP/s).  128 x 128: 5003 f16 rows over 60 groups 1410 x 2048 in 98 us, bound by the weights'
// 346 MB (3.8 TB/s) with two K-steps in flight per unit.  64 x 64, four stages: 2048 bf16 rows over 64 groups 1408 x 2048
// in 77 us (4.9 TB/s); int8 128 x 4096 x 4096 13.3 us, 25.5 with two stages.
template <int DT, int BM, int BN, int WM, int WN, int LA, int LB, int RB, int STAGES, typename Params>
__device__ __forceinline__ void token_tile_dl(const void *a, const void *b, void *c, const void *bias, const Params &q,
                                              int tm, int tn, int part, int parts) {
  if constexpr (BM == 256) {
    static_assert(BN == 256 && WM == 2 && WN == 4 && STAGES == 2, "the parts below");
    using L = DlLds<DT, BM, BN, RB, LA, LB, 2>;
    __shared__ __attribute__((aligned(1024))) char lds[L::FIRST];
    __shared__ __attribute__((aligned(1024))) char lds_hi[L::KM ? L::STAGE : 1024];
    const int m0 = tm * 256, n0 = tn * 256;
    if (parts == 1) {
      contraction_tile_in<DT, 256, 256, 2, 4, RB, LA, LB, false, 2>(a, b, c, bias, nullptr, q, 0, m0, n0, lds, lds_hi,
                                                                    nullptr, nullptr);
      return;
    }
    const int m = m0 + (part & 1) * 128, n = n0 + (part >> 1) * 128;
    if (m >= q.M || n >= q.N)
      return;
    if (parts == 2)
      contraction_tile_in<DT, 128, 256, 2, 4, RB, LA, LB, false, 2>(a, b, c, bias, nullptr, q, 0, m, n, lds, lds_hi,
                                                                    nullptr, nullptr);
    else
      contraction_tile_in<DT, 128, 128, 2, 4, RB, LA, LB, false, 2>(a, b, c, bias, nullptr, q, 0, m, n, lds, lds_hi,
                                                                    nullptr, nullptr);
  } else {
    contraction_tile_dl<DT, BM, BN, WM, WN, RB, LA, LB, false, STAGES>(a, b, c, bias, nullptr, q, 0, tm * BM, tn * BN);
  }
}

template <int DT, int BM, int BN, int WM, int WN, int LB, int RB, int STAGES>
__device__ __forceinline__ void token_gemm_body_dl(const void *A, const void *B, void *C, const void *bias,
                                                   const int32_t *offsets, const float *token_scale,
                                                   const float *channel_scale, const RockTokenGemmParams &tp) {
  GroupTile t;
  if (!locate_tile<BM, BM == 256>(offsets, tp.gemm, t))
    return;
  with_group<DT>(A, B, C, bias, token_scale, channel_scale, tp, t,
                 [&](const void *a, const void *b, void *c, const void *x, const auto &q) __attribute__((always_inline)) {
                   token_tile_dl<DT, BM, BN, WM, WN, LD_ROWS_FAST, LB, RB, STAGES>(a, b, c, x, q, t.tm, t.tn, t.part,
                                                                                   t.parts);
                 });
}

// ---- operands of any alignment -----------------------------------------------------------------
// Tiles of rows that are not whole 16-byte chunks: global -> registers -> LDS, the loads of the next AHEAD K-steps in
// flight while one is multiplied, LDS as in the other tile kernels.  Every load is 16 bytes from wherever they start
// (global loads need no alignment; off 4-byte boundaries they run at about half the aligned rate): a chunk that would run
// past the end of its row is loaded from that many elements further down and moved into place on its way to LDS, which
// fills it up with zeros.  Rows behind the last are read as the last one, their products are not stored.
// Rows shorter than a chunk are loaded element by element.
// Measured on MI355X: int8 1001 x 2307 x 1283 19 us (1280 deep on the aligned 64 x 64 tiles 13, 1284 deep here 15, so four of
// the six are the loads' alignment), 4000 x 4096 x 2051 on 128 x 128 tiles 94.  Rows of 1410 f16 start on 4-byte boundaries
// and lose elsewhere: with three K-steps in registers a 128 x 128 wave takes 318 of them (190 and 128 accumulation
// registers) and its block a unit to itself, where the aligned weight gradient runs three a unit.  60 groups 1410 x 2048 at
// 5003 rows: gradient of the rows 118 us, of the weights 235 (1408 columns on the aligned kernels: 97 and 99).
__device__ __forceinline__ v4i move_down(const v4i &v, int bytes) { // byte i <- byte i + bytes, zeros from behind
  typedef uint64_t v2u __attribute__((ext_vector_type(2)));
  const v2u w = __builtin_bit_cast(v2u, v);
  const int bits = bytes * 8;
  v2u r;
  r[0] = bits == 0 ? w[0] : bits < 64 ? (w[0] >> bits) | (w[1] << (64 - bits)) : bits < 128 ? w[1] >> (bits - 64) : 0;
  r[1] = bits < 64 ? w[1] >> bits : 0;
  return __builtin_bit_cast(v4i, r);
}

// The chunk of elements k .. of a row whose element k lies at src, as zeros from element K on.  Every lane loads all its
// elements, those behind the last as the last: loads behind a test each would wait for each other, sixteen times the
// latency of memory.
template <int DT> __device__ __forceinline__ v4i tail_chunk(const char *src, int k, int K) {
  constexpr int ES = MmaTraits<DT>::ES;
  uint32_t v[kChunk / ES];
#pragma unroll
  for (int e = 0; e < kChunk / ES; ++e)
    v[e] = load_elem<ES>(src, min(e, K - 1 - k));
  return gather_chunk<DT>([&](int e) { return k + e < K ? v[e] : 0u; });
}

// K-contiguous rows
template <int DT, int ROWS, int NT> struct AnyRows {
  using Gm = TileGeom<DT, ROWS, NT>;
  const char *row[Gm::NCH];
  int k0, K, tid;
  __device__ __forceinline__ void init(const void *base, int64_t row_stride, int64_t, int row0, int rows, int K_, int t) {
    tid = t;
    K = K_;
    k0 = (t & 7) * Gm::EPC;
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i)
      row[i] = (const char *)base + (int64_t)min(row0 + (t >> 3) + i * Gm::ROW_STEP, rows - 1) * row_stride * Gm::ES;
  }
  static __device__ __forceinline__ bool narrow(int K, int) { return K < Gm::EPC; }
  __device__ __forceinline__ void load(int kt, v4i (&r)[Gm::NCH]) const {
    const int k = min(kt * Gm::BKE + k0, K - Gm::EPC);
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i)
      __builtin_memcpy(&r[i], row[i] + (int64_t)k * Gm::ES, 16);
  }
  __device__ __forceinline__ void load_elements(int kt, v4i (&r)[Gm::NCH]) const {
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i)
      r[i] = tail_chunk<DT>(row[i] + (int64_t)(kt * Gm::BKE + k0) * Gm::ES, kt * Gm::BKE + k0, K);
  }
  // last: K-step kt may hold the end of the rows
  __device__ __forceinline__ void store(int kt, bool last, char *lds, v4i (&r)[Gm::NCH]) const {
    if (last) {
      const int k = kt * Gm::BKE + k0, beyond = k - min(k, K - Gm::EPC);
#pragma unroll
      for (int i = 0; i < Gm::NCH; ++i)
        r[i] = move_down(r[i], min(beyond, Gm::EPC) * Gm::ES);
    }
    store_tile<DT, ROWS, NT>(lds, r, tid);
  }
  __device__ __forceinline__ void store_elements(char *lds, const v4i (&r)[Gm::NCH]) const { store_tile<DT, ROWS, NT>(lds, r, tid); }
  static __device__ __forceinline__ Frag<DT> fragment(const char *lds, int block, int step, int lane) {
    return read_frag<DT>(lds, block + (lane & 31), step, lane >> 5);
  }
};

// K-major columns: 16 bytes of consecutive columns of one k per load, LDS as ColsDl fills it (k-rows of swizzled chunks,
// turned by the transposing reads)
template <int DT, int COLS, int NT> struct AnyCols {
  using Kg = KmGeom<DT, COLS, kRowBytes>;
  struct Gm {
    static constexpr int ES = Kg::ES, EPC = kChunk / ES, NCH = COLS * kRowBytes / kChunk / NT;
    static_assert(COLS * kRowBytes % (kChunk * NT) == 0, "whole chunks per thread");
  };
  const char *base; // the tile's first column
  int64_t pitch;    // bytes between consecutive k
  // byte where a lane's chunk is loaded from, counted from the tile's first column (rows may be longer than 2 GiB; a
  // chunk moved back from the row's end may start in front of the tile), elements it is moved down by
  int at[Gm::NCH], beyond[Gm::NCH];
  int first, cols, K, tid;
  bool edge; // some lane's chunk is moved
  __device__ __forceinline__ void init(const void *b, int64_t, int64_t ks, int col0, int c, int K_, int t) {
    base = (const char *)b + (int64_t)col0 * Gm::ES;
    pitch = ks * Gm::ES;
    first = col0;
    cols = c;
    K = K_;
    tid = t;
    edge = col0 + COLS > c;
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i) {
      const int col = col0 + (((t + i * NT) % Kg::CPR) ^ Kg::swz(krow(i))) * Gm::EPC, from = max(min(col, c - Gm::EPC), 0);
      at[i] = (from - col0) * Gm::ES;
      beyond[i] = min(col - from, Gm::EPC);
    }
  }
  __device__ __forceinline__ int krow(int i) const { return (tid + i * NT) / Kg::CPR; }
  static __device__ __forceinline__ bool narrow(int, int cols) { return cols < Gm::EPC; }
  __device__ __forceinline__ const char *row(int kt, int i) const {
    return base + (int64_t)min(kt * Kg::KR + krow(i), K - 1) * pitch;
  }
  __device__ __forceinline__ void load(int kt, v4i (&r)[Gm::NCH]) const {
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i)
      __builtin_memcpy(&r[i], row(kt, i) + at[i], 16);
  }
  __device__ __forceinline__ void load_elements(int kt, v4i (&r)[Gm::NCH]) const {
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i) {
      r[i] = tail_chunk<DT>(row(kt, i) + at[i] + beyond[i] * Gm::ES, first + at[i] / Gm::ES + beyond[i], cols);
      if (kt * Kg::KR + krow(i) >= K)
        r[i] = v4i{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ void store(int kt, bool last, char *lds, v4i (&r)[Gm::NCH]) const {
    if (edge) {
#pragma unroll
      for (int i = 0; i < Gm::NCH; ++i)
        r[i] = move_down(r[i], beyond[i] * Gm::ES);
    }
    if (last) {
#pragma unroll
      for (int i = 0; i < Gm::NCH; ++i)
        r[i] = kt * Kg::KR + krow(i) < K ? r[i] : v4i{0, 0, 0, 0};
    }
    store_elements(lds, r);
  }
  __device__ __forceinline__ void store_elements(char *lds, const v4i (&r)[Gm::NCH]) const {
#pragma unroll
    for (int i = 0; i < Gm::NCH; ++i)
      *(v4i *)(lds + (tid + i * NT) * kChunk) = r[i];
  }
  static __device__ __forceinline__ Frag<DT> fragment(const char *lds, int block, int step, int lane) {
    return dl_read_frag_km<DT, COLS, kRowBytes>(lds, block, step, lane);
  }
};

template <int DT, int BM, int BN, int WM, int WN, int AHEAD, typename LoadA, typename LoadB, typename Params>
__device__ __forceinline__ void any_tile(const void *A, const void *B, void *C, const void *bias, const Params &p, int m0,
                                         int n0) {
  using Tr = MmaTraits<DT>;
  using Acc = typename Tr::Acc;
  constexpr int WTM = BM / WM, WTN = BN / WN, MI = WTM / 32, NI = WTN / 32, NW = WM * WN;
  constexpr int STEPS = kChunksPerRow / (2 * Tr::CHUNKS), BKE = kRowBytes / Tr::ES;
  constexpr int A_BYTES = BM * kRowBytes, STAGE = A_BYTES + BN * kRowBytes;
  __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  LoadA la;
  LoadB lb;
  la.init(A, p.a_ms, p.a_ks, m0, p.M, p.K, tid);
  lb.init(B, p.b_ns, p.b_ks, n0, p.N, p.K, tid);
  v4i ra[AHEAD][LoadA::Gm::NCH], rb[AHEAD][LoadB::Gm::NCH];
  Acc acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        acc[i][j][v] = 0;
  const int nk = (p.K + BKE - 1) / BKE;
  int stage = 0;
  // Two stages, one barrier: when everyone has passed the barrier of a step, everyone is done with the step before it,
  // whose stage the next one overwrites.
  auto multiply = [&]() __attribute__((always_inline)) {
    const char *sa = lds + stage * STAGE, *sb = sa + A_BYTES;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      Frag<DT> fb[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j)
        fb[j] = LoadB::fragment(sb, wn * WTN + j * 32, s, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const Frag<DT> fa = LoadA::fragment(sa, wm * WTM + i * 32, s, lane);
#pragma unroll
        for (int j = 0; j < NI; ++j)
          mma32x32<DT>(fb[j], fa, acc[i][j]);
      }
    }
    stage ^= 1;
  };
  if (LoadA::narrow(p.K, p.M) || LoadB::narrow(p.K, p.N)) {
    for (int kt = 0; kt < nk; ++kt) {
      la.load_elements(kt, ra[0]);
      lb.load_elements(kt, rb[0]);
      la.store_elements(lds + stage * STAGE, ra[0]);
      lb.store_elements(lds + stage * STAGE + A_BYTES, rb[0]);
      multiply();
    }
  } else if (nk > 0) {
    // (behind the last K-step the last one is loaded again, so that the loop needs no branch around its loads)
    auto fetch = [&](int kt, v4i(&a)[LoadA::Gm::NCH], v4i(&b)[LoadB::Gm::NCH]) __attribute__((always_inline)) {
      la.load(min(kt, nk - 1), a);
      lb.load(min(kt, nk - 1), b);
    };
    auto to_lds = [&](int kt, v4i(&a)[LoadA::Gm::NCH], v4i(&b)[LoadB::Gm::NCH]) __attribute__((always_inline)) {
      la.store(kt, kt == nk - 1, lds + stage * STAGE, a);
      lb.store(kt, kt == nk - 1, lds + stage * STAGE + A_BYTES, b);
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
      fetch(s, ra[s], rb[s]);
    int kt = 0;
    for (; kt + AHEAD <= nk; kt += AHEAD)
      static_for<AHEAD>([&](auto sc) __attribute__((always_inline)) {
        constexpr int s = decltype(sc)::value;
        to_lds(kt + s, ra[s], rb[s]);
        fetch(kt + s + AHEAD, ra[s], rb[s]);
        multiply();
      });
    static_for<AHEAD>([&](auto sc) __attribute__((always_inline)) {
      constexpr int s = decltype(sc)::value;
      if (kt + s < nk) {
        to_lds(kt + s, ra[s], rb[s]);
        multiply();
      }
    });
  }
  if constexpr (HasRowScales<Params>::value)
    row_scale_epilogue<DT, MI, NI, NW, 2 * STAGE>(acc, p, 0, C, bias, m0 + wm * WTM, n0 + wn * WTN, lds, wave, lane);
  else
    dl_epilogue<DT, MI, NI, NW, 2 * STAGE>(acc, p, 0, C, bias, nullptr, m0 + wm * WTM, n0 + wn * WTN, lds, wave, lane);
}

// B_COLS: the weights are stored [depth, columns]
template <int DT, int BM, int BN, int WM, int WN, bool B_COLS>
__device__ __forceinline__ void token_gemm_body_any(const void *A, const void *B, void *C, const void *bias,
                                                    const int32_t *offsets, const float *token_scale,
                                                    const float *channel_scale, const RockTokenGemmParams &tp) {
  constexpr int NT = WM * WN * 64;
  GroupTile t;
  if (!locate_tile<BM>(offsets, tp.gemm, t))
    return;
  with_group<DT>(A, B, C, bias, token_scale, channel_scale, tp, t,
                 [&](const void *a, const void *b, void *c, const void *x, const auto &q) __attribute__((always_inline)) {
                   using LoadB = std::conditional_t<B_COLS, AnyCols<DT, BN, NT>, AnyRows<DT, BN, NT>>;
                   any_tile<DT, BM, BN, WM, WN, 3, AnyRows<DT, BM, NT>, LoadB>(a, b, c, x, q, t.tm * BM, t.tn * BN);
                 });
}

// ---- few rows ------------------------------------------------------------------------------------
// Products of a few token rows are bound by the weights' bytes, and what a tile kernel spends on filling LDS for one or
// two K-steps at a time is latency.  Here a block takes 16 * CT columns and 16 * MT rows, its eight waves divide the
// depth (64 bytes of every row in turn), weights and rows go straight from global memory into the operands of the 16 x 16
// matrix instructions -- each weight is used by one wave only, so LDS has nothing to share -- with UNROLL K-steps of loads
// in flight per wave, and the partial sums of the waves are added in wave order through LDS.
template <int DT> struct SmallMma; // acc[n = 4 * (lane / 16) + v][m = lane % 16] += 16 bytes of k per lane and operand
template <> struct SmallMma<MM_I8> {
  using Acc = v4i;
  static __device__ __forceinline__ Acc step(const v4i &w, const v4i &x, const Acc &c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
  }
};
template <> struct SmallMma<MM_F16> {
  using Acc = v4f;
  static __device__ __forceinline__ Acc step(const v4i &w, const v4i &x, const Acc &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w), __builtin_bit_cast(v8h, x), c, 0, 0, 0);
  }
};
template <> struct SmallMma<MM_BF16> {
  using Acc = v4f;
  static __device__ __forceinline__ Acc step(const v4i &w, const v4i &x, const Acc &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, w), __builtin_bit_cast(v8bf, x), c, 0, 0, 0);
  }
};
template <> struct SmallMma<MM_F32> {
  using Acc = v4f;
  static __device__ __forceinline__ Acc step(const v4i &w, const v4i &x, Acc c) {
    const v4f a = __builtin_bit_cast(v4f, w), b = __builtin_bit_cast(v4f, x);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
};

constexpr int kSkinnyWaves = 8;

template <int DT, int MT, int CT, int UNROLL, typename Params>
__device__ __forceinline__ void skinny_tile(const void *A, const void *B, void *C, const void *bias, const Params &p,
                                            int m0, int n0) {
  using Mma = SmallMma<DT>;
  using Acc = typename Mma::Acc;
  constexpr int ES = MmaTraits<DT>::ES, EPC = kChunk / ES, STEP = 64 / ES, W = kSkinnyWaves;
  __shared__ __attribute__((aligned(16))) char lds[W * MT * CT * 64 * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, slice = lane >> 4;
  const char *w[CT], *x[MT]; // rows behind the last are read as the last one: their results are not stored
#pragma unroll
  for (int j = 0; j < CT; ++j)
    w[j] = (const char *)B + (int64_t)min(n0 + j * 16 + l16, p.N - 1) * p.b_ns * ES;
#pragma unroll
  for (int i = 0; i < MT; ++i)
    x[i] = (const char *)A + (int64_t)min(m0 + i * 16 + l16, p.M - 1) * p.a_ms * ES;
  Acc acc[MT][CT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
      acc[i][j] = Acc{0, 0, 0, 0};

  const int steps = p.K / STEP; // whole K-steps: 64 bytes of every row
  int s = wave;
  auto batch = [&](auto n_const) __attribute__((always_inline)) {
    constexpr int U = decltype(n_const)::value;
    v4i wr[U][CT], xr[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = ((int64_t)(s + u * W) * 4 + slice) * kChunk;
#pragma unroll
      for (int j = 0; j < CT; ++j)
        __builtin_memcpy(&wr[u][j], w[j] + at, 16);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        __builtin_memcpy(&xr[u][i], x[i] + at, 16);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j)
          acc[i][j] = Mma::step(wr[u][j], xr[u][i], acc[i][j]);
    s += U * W;
  };
  while (s + (UNROLL - 1) * W < steps)
    batch(std::integral_constant<int, UNROLL>{});
  if (UNROLL > 4 && s + 3 * W < steps)
    batch(std::integral_constant<int, 4>{});
  if (UNROLL > 2 && s + W < steps)
    batch(std::integral_constant<int, 2>{});
  if (s < steps)
    batch(std::integral_constant<int, 1>{});
  if (steps * STEP < p.K && wave == steps % W) { // what is left of K, less than a step
    const int k = steps * STEP + slice * EPC;
    v4i wr[CT], xr[MT];
#pragma unroll
    for (int j = 0; j < CT; ++j)
      wr[j] = tail_chunk<DT>(w[j] + (int64_t)k * ES, k, p.K);
#pragma unroll
    for (int i = 0; i < MT; ++i)
      xr[i] = tail_chunk<DT>(x[i] + (int64_t)k * ES, k, p.K);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j)
        acc[i][j] = Mma::step(wr[j], xr[i], acc[i][j]);
  }

  Acc *sums = (Acc *)lds; // [wave][tile][lane]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
      sums[(wave * MT * CT + i * CT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  static_assert(MT * CT <= W, "a wave finishes one tile");
  if (wave >= MT * CT)
    return;
  Acc sum = sums[wave * 64 + lane];
#pragma unroll
  for (int o = 1; o < W; ++o)
    sum += sums[(o * MT * CT + wave) * 64 + lane];
  const int m = m0 + wave / CT * 16 + l16, n = n0 + wave % CT * 16 + slice * 4;
  if (m >= p.M || n >= p.N)
    return;
  int64_t row_off, n_stride;
  bool vec_ok;
  out_row_addr(p, 0, m, C, row_off, n_stride, vec_ok);
  dispatch_tile_dtype<MmaTraits<DT>::INT_ACC>(p, [&](auto od_const) __attribute__((always_inline)) {
    constexpr int OD = decltype(od_const)::value;
    const v4i raw = token_convert4<OD>(sum, p, m, bias, n);
    store_packed4(raw, OutElemSize<OD>::value, C, row_off + n, n_stride, n, p.N, vec_ok);
  });
}

template <int DT, int MT, int CT, int UNROLL>
__device__ __forceinline__ void token_gemm_body_skinny(const void *A, const void *B, void *C, const void *bias,
                                                       const int32_t *offsets, const float *token_scale,
                                                       const float *channel_scale, const RockTokenGemmParams &tp) {
  GroupTile t;
  if (!locate_tile<MT * 16>(offsets, tp.gemm, t))
    return;
  with_group<DT>(A, B, C, bias, token_scale, channel_scale, tp, t,
                 [&](const void *a, const void *b, void *c, const void *x, const auto &q) __attribute__((always_inline)) {
                   skinny_tile<DT, MT, CT, UNROLL>(a, b, c, x, q, t.tm * MT * 16, t.tn * CT * 16);
                 });
}

// ---- weight gradient -----------------------------------------------------------------------
// C[e] = sum over the group's rows of A^T B, both operands K-major.  Long reductions are bound by the matrix cores (16384
// bf16 rows over 8 groups, 4096 x 2048 results: 230 us, 1.19 PFLOP/s on 256 x 256 tiles), short ones by their results (60
// groups 1408 x 2048 at 83 rows: 92 us for 346 MB on 128 x 128 tiles, three of them per unit).
// (its own type: the loaders below instead of those for operands within one 2 GiB window; results of the operands' type,
// so that a wave's staging region takes half the LDS for 16-bit ones)
template <int DT> struct TokenWeightTile : TokenTileParams {};
template <int DT> struct AnyRowStart<TokenWeightTile<DT>> : std::true_type {};
template <int DT> struct MaxOutBytes<TokenWeightTile<DT>, DT> : std::integral_constant<int, MmaTraits<DT>::ES> {};
template <bool INT_ACC, int DT, typename F>
__device__ __forceinline__ void dispatch_tile_dtype(const TokenWeightTile<DT> &, F &&f) {
  f(std::integral_constant<int, DT>{});
}

// ColsDl for a reduction over any number of rows: the buffer descriptor's base moves on with the K-steps in 64 bits
// (scalar additions) and the lanes' offsets stay inside one stage.
template <int DT, int COLS, int NW, int RB> struct ColsLongDl {
  using Kg = KmGeom<DT, COLS, RB>;
  struct Sg {
    static constexpr int SLABS = COLS * RB / 1024;
    static constexpr int PER_WAVE = SLABS / NW;
    static_assert(SLABS % NW == 0, "stage must split into 1 KiB slabs per wave");
  };
  static constexpr int ES = Kg::ES;
  const char *base;
  int64_t step_bytes;         // between K-steps
  unsigned off[Sg::PER_WAVE]; // byte offset of this lane's chunk inside a K-step, or kOobOffset
  int krow[Sg::PER_WAVE];     // k-row of the chunk inside a stage
  int K;
  int wave;

  __device__ __forceinline__ void init(const void *b, int64_t k_stride, int col0, int cols_total, int K_, int wave_,
                                       int lane) {
    wave = wave_;
    K = K_;
    base = (const char *)b + (int64_t)col0 * ES;
    step_bytes = k_stride * ES * Kg::KR;
#pragma unroll
    for (int i = 0; i < Sg::PER_WAVE; ++i) {
      const int idx = (wave * Sg::PER_WAVE + i) * 64 + lane; // physical chunk inside the stage
      const int r = idx / Kg::CPR, pc = idx % Kg::CPR;
      const int lc = pc ^ Kg::swz(r); // logical chunk this lane fetches
      krow[i] = r;
      const bool col_ok = col0 + (lc + 1) * (kChunk / ES) <= cols_total;
      off[i] = col_ok ? (unsigned)(r * (int)k_stride * ES + lc * kChunk) : kOobOffset;
    }
  }
  __device__ __forceinline__ void issue(int kt, char *stage) {
    const __amdgpu_buffer_rsrc_t rsrc = dl_rsrc(base + kt * step_bytes);
    const int k0 = kt * Kg::KR;
#pragma unroll
    for (int i = 0; i < Sg::PER_WAVE; ++i) {
      const unsigned voff = (k0 + krow[i] < K) ? off[i] : kOobOffset;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (lds_void_t *)(stage + (wave * Sg::PER_WAVE + i) * 1024), 16, (int)voff, 0, 0, 0);
    }
  }
};
template <int DT, int ROWS, int NW, int RB, int KIND>
__device__ __forceinline__ auto make_dl_a(const void *A, const TokenWeightTile<DT> &p, int, int m0, int wave, int lane) {
  ColsLongDl<DT, ROWS, NW, RB> l;
  l.init(A, p.a_ks, m0, p.M, p.K, wave, lane);
  return l;
}
template <int DT, int ROWS, int NW, int RB, int KIND>
__device__ __forceinline__ auto make_dl_b(const void *B, const TokenWeightTile<DT> &p, int, int n0, int wave, int lane) {
  ColsLongDl<DT, ROWS, NW, RB> l;
  l.init(B, p.b_ks, n0, p.N, p.K, wave, lane);
  return l;
}

// Group g's rows among M, as scan_groups reads the boundaries: from the furthest one up to the group's own, so that the
// gradient sums exactly the rows that the product gave to the group.  Uniform over the block.  `mine`: the lane's boundary
// of the first 64, loaded before the block has worked out its tile (64 groups 768 x 1024 at 16 rows, three rounds of blocks:
// 26.7 us, 27.5 loaded afterwards).
__device__ __forceinline__ int lane_boundary(const int32_t *offsets, int G) { return offsets[min((int)(threadIdx.x & 63), G)]; }
__device__ __forceinline__ void group_rows(const int32_t *offsets, int mine, int g, int M, int &row0, int &rows) {
  const int lane = threadIdx.x & 63;
  int own, next, top = lane <= g ? mine : 0;
  if (g < 63) {
    own = __builtin_amdgcn_readlane(mine, g);
    next = __builtin_amdgcn_readlane(mine, g + 1);
  } else {
    own = offsets[g];
    next = offsets[g + 1];
    for (int base = 64; base <= g; base += 64)
      top = max(top, offsets[min(base + lane, g)]);
  }
  if (__builtin_amdgcn_ballot_w64(top > own)) { // some boundary before it lies further on (or this one below 0)
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = lane_value(top, lane ^ d);
      top = max(top, other);
    }
  } else {
    top = own;
  }
  row0 = __builtin_amdgcn_readfirstlane(min(max(top, 0), M));
  rows = __builtin_amdgcn_readfirstlane(min(max(next, row0), M)) - row0;
}

// Group g's rows as the reduction: operands and result moved to the group, gemm.K its number of rows
template <int DT, typename F>
__device__ __forceinline__ void with_weight_group(const void *A, const void *B, void *C, const int32_t *offsets,
                                                  int mine, const RockTokenWeightParams &wp, int g, F &&f) {
  constexpr int ES = MmaTraits<DT>::ES;
  TokenWeightTile<DT> q;
  static_cast<RockGemmParams &>(q) = wp.gemm;
  int first, rows;
  group_rows(offsets, mine, g, q.K, first, rows);
  q.K = rows;
  const int64_t row0 = first;
  f((const char *)A + row0 * q.a_ks * ES, (const char *)B + row0 * q.b_ks * ES,
    (char *)C + (int64_t)g * q.c_gs * token_out_size(q.epi.out_dtype), q);
}

// Group by group: the tiles of one group go round the XCDs, so that a group with more rows than the others keeps all of
// them busy longer and not the one that holds it.
template <bool SPLIT>
__device__ __forceinline__ bool locate_weight_tile(const RockGemmParams &p, GroupTile &t) {
  int id;
  const int tiles = p.tiles_m * p.tiles_n;
  if (!block_tile<SPLIT>(tiles * p.G, false, id, t.part, t.parts))
    return false;
  t.e = id / tiles;
  const int in_group = id - t.e * tiles;
  const int group_sz = p.group_m * p.tiles_n;
  const int grp = in_group / group_sz;
  const int first_m = grp * p.group_m;
  const int rows_here = min(p.tiles_m - first_m, p.group_m);
  const int in_grp = in_group - grp * group_sz;
  t.tm = first_m + in_grp % rows_here;
  t.tn = in_grp / rows_here;
  return true;
}

template <int DT, int BM, int BN, int WM, int WN, int RB, int STAGES>
__device__ __forceinline__ void token_weight_body_dl(const void *A, const void *B, void *C, const int32_t *offsets,
                                                     const RockTokenWeightParams &wp) {
  const int mine = lane_boundary(offsets, wp.gemm.G);
  GroupTile t;
  if (!locate_weight_tile<BM == 256>(wp.gemm, t))
    return;
  with_weight_group<DT>(A, B, C, offsets, mine, wp, t.e,
                        [&](const void *a, const void *b, void *c, const TokenWeightTile<DT> &q)
                            __attribute__((always_inline)) {
                              token_tile_dl<DT, BM, BN, WM, WN, LD_COLS_FAST, LD_COLS_FAST, RB, STAGES>(
                                  a, b, c, nullptr, q, t.tm, t.tn, t.part, t.parts);
                            });
}

// Few results with a long reduction: a 64 x 64 tile by sixteen waves, four groups of four that take a quarter of the rows
// each on LDS stages of their own; their sums are added in group order through LDS.  The reduction of a block is a chain
// of memory latencies, one per K-step, and this chain is a quarter as long (each step takes more than twice as long, with
// four times the loads to wait for): one 512 x 512 result of 4000 bf16 rows 23 us on MI355X, 34 by four waves a block.
template <int DT>
__device__ __forceinline__ void token_weight_body_split(const void *A, const void *B, void *C, const int32_t *offsets,
                                                        const RockTokenWeightParams &wp) {
  using Acc = typename MmaTraits<DT>::Acc;
  constexpr int RB = 128, T = 64, SPLIT = 4, ES = MmaTraits<DT>::ES, KR = RB / ES, STEPS = kChunksPerRow / 2;
  constexpr int A_BYTES = T * RB, STAGE = 2 * A_BYTES;
  // one LDS object per stage, see DlLds
  __shared__ __attribute__((aligned(1024))) char lds[SPLIT * STAGE];
  __shared__ __attribute__((aligned(1024))) char lds_hi[SPLIT * STAGE];
  const int mine = lane_boundary(offsets, wp.gemm.G);
  GroupTile t;
  if (!locate_weight_tile<false>(wp.gemm, t))
    return;
  const int lane = threadIdx.x & 63, all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int share = all >> 2, wave = all & 3, wm = wave & 1, wn = wave >> 1;
  with_weight_group<DT>(A, B, C, offsets, mine, wp, t.e, [&](const void *a, const void *b, void *c, const TokenWeightTile<DT> &q)
                                                       __attribute__((always_inline)) {
    ColsLongDl<DT, T, 4, RB> la, lb;
    la.init(a, q.a_ks, t.tm * T, q.M, q.K, wave, lane);
    lb.init(b, q.b_ks, t.tn * T, q.N, q.K, wave, lane);
    Acc acc[1][1];
#pragma unroll
    for (int v = 0; v < 16; ++v)
      acc[0][0][v] = 0;
    const int nk = (q.K + KR - 1) / KR, per = (nk + SPLIT - 1) / SPLIT;
    // K-step i of this share; steps behind the share or the reduction load zeros
    auto issue = [&](int i, char *stage) __attribute__((always_inline)) {
      const int kt = i < per ? share * per + i : nk;
      la.issue(kt, stage + share * STAGE);
      lb.issue(kt, stage + share * STAGE + A_BYTES);
    };
    auto kstep = [&](int i, const char *stage, char *refill) __attribute__((always_inline)) {
      stage += opaque_zero(); // (see contraction_tile_in)
      wait_vmcnt_and_lds_reads<0>();
      __builtin_amdgcn_s_barrier();
      issue(i + 1, refill);
      const char *sa = stage + share * STAGE, *sb = sa + A_BYTES;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const Frag<DT> fb = dl_read_frag_km<DT, T, RB>(sb, wn * 32, s, lane);
        const Frag<DT> fa = dl_read_frag_km<DT, T, RB>(sa, wm * 32, s, lane);
        mma32x32<DT>(fb, fa, acc[0][0]);
      }
    };
    issue(0, lds);
    int i = 0;
    for (; i + 1 < per; i += 2) {
      kstep(i, lds, lds_hi);
      kstep(i + 1, lds_hi, lds);
    }
    if (i < per)
      kstep(i, lds, lds_hi);
    wait_vmcnt_and_lds_reads<0>();
    __builtin_amdgcn_s_barrier(); // no load into LDS and no read of a stage is left
    typedef float sums_t __attribute__((ext_vector_type(4)));
    sums_t *sums = (sums_t *)lds_hi;
    static_assert((SPLIT - 1) * 4 * 4 * 64 * 16 <= SPLIT * STAGE, "the shares' sums fit in the stages");
    if (share > 0) {
#pragma unroll
      for (int v = 0; v < 4; ++v)
        sums[(((share - 1) * 4 + wave) * 4 + v) * 64 + lane] =
            sums_t{acc[0][0][4 * v], acc[0][0][4 * v + 1], acc[0][0][4 * v + 2], acc[0][0][4 * v + 3]};
    }
    __syncthreads();
    if (share > 0) {
      __builtin_amdgcn_s_barrier(); // the one in dl_epilogue
      return;
    }
#pragma unroll
    for (int o = 0; o < SPLIT - 1; ++o)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const sums_t x = sums[((o * 4 + wave) * 4 + v) * 64 + lane];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          acc[0][0][4 * v + k] = acc[0][0][4 * v + k] + x[k];
      }
    dl_epilogue<DT, 1, 1, 4, SPLIT * STAGE>(acc, q, 0, c, nullptr, nullptr, t.tm * T + wm * 32, t.tn * T + wn * 32, lds,
                                            wave, lane);
  });
}

template <int DT, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void token_weight_body_any(const void *A, const void *B, void *C, const int32_t *offsets,
                                                      const RockTokenWeightParams &wp) {
  constexpr int NT = WM * WN * 64;
  const int mine = lane_boundary(offsets, wp.gemm.G);
  GroupTile t;
  if (!locate_weight_tile<false>(wp.gemm, t))
    return;
  with_weight_group<DT>(A, B, C, offsets, mine, wp, t.e,
                        [&](const void *a, const void *b, void *c, const TokenWeightTile<DT> &q)
                            __attribute__((always_inline)) {
                              any_tile<DT, BM, BN, WM, WN, 3, AnyCols<DT, BM, NT>, AnyCols<DT, BN, NT>>(
                                  a, b, c, nullptr, q, t.tm * BM, t.tn * BN);
                            });
}

} // namespace rk

// ---- kernel-defining macros (rocmlir_amd/_build.py holds the list of kernels) -----------------
#define RK_TG_CAT_(a, b) a##b
#define RK_TG_CAT(a, b) RK_TG_CAT_(a, b)
#define RK_TOKEN_GEMM_NAME(NAME) RK_TG_CAT(RK_TG_CAT(rock_token_gemm_, ROCK_DTNAME), NAME)
#define RK_TOKEN_WEIGHT_NAME(NAME) RK_TG_CAT(RK_TG_CAT(rock_token_gemm_bwd_weight_, ROCK_DTNAME), NAME)
#define RK_TOKEN_GEMM_ARGS                                                                            \
  const void *A, const void *B, void *C, const void *bias, const int32_t *offsets,                    \
      const float *token_scale, const float *channel_scale, RockTokenGemmParams p

#define RK_TOKEN_GEMM_DL(NAME, BM, BN, WM, WN, LB, RB, STAGES)                                        \
  extern "C" __global__ __launch_bounds__(WM *WN * 64) void RK_TOKEN_GEMM_NAME(NAME)(RK_TOKEN_GEMM_ARGS) { \
    rk::token_gemm_body_dl<ROCK_DT, BM, BN, WM, WN, LB, RB, STAGES>(A, B, C, bias, offsets, token_scale, channel_scale, p); \
  }
#define RK_TOKEN_GEMM_ANY(NAME, BM, BN, WM, WN, B_COLS)                                               \
  extern "C" __global__ __launch_bounds__(WM *WN * 64) void RK_TOKEN_GEMM_NAME(NAME)(RK_TOKEN_GEMM_ARGS) { \
    rk::token_gemm_body_any<ROCK_DT, BM, BN, WM, WN, B_COLS>(A, B, C, bias, offsets, token_scale, channel_scale, p); \
  }
#define RK_TOKEN_GEMM_SKINNY(NAME, MT, CT, UNROLL)                                                    \
  extern "C" __global__ __launch_bounds__(512) void RK_TOKEN_GEMM_NAME(NAME)(RK_TOKEN_GEMM_ARGS) {     \
    rk::token_gemm_body_skinny<ROCK_DT, MT, CT, UNROLL>(A, B, C, bias, offsets, token_scale, channel_scale, p); \
  }
#define RK_TOKEN_WEIGHT_DL(NAME, BM, BN, WM, WN, RB, STAGES)                                          \
  extern "C" __global__ __launch_bounds__(WM *WN * 64) void RK_TOKEN_WEIGHT_NAME(NAME)(               \
      const void *A, const void *B, void *C, const int32_t *offsets, RockTokenWeightParams p) {       \
    rk::token_weight_body_dl<ROCK_DT, BM, BN, WM, WN, RB, STAGES>(A, B, C, offsets, p);                           \
  }
#define RK_TOKEN_WEIGHT_SPLIT(NAME)                                                                   \
  extern "C" __global__ __launch_bounds__(1024) void RK_TOKEN_WEIGHT_NAME(NAME)(                      \
      const void *A, const void *B, void *C, const int32_t *offsets, RockTokenWeightParams p) {       \
    rk::token_weight_body_split<ROCK_DT>(A, B, C, offsets, p);                                        \
  }
#define RK_TOKEN_WEIGHT_ANY(NAME, BM, BN, WM, WN)                                                     \
  extern "C" __global__ __launch_bounds__(WM *WN * 64) void RK_TOKEN_WEIGHT_NAME(NAME)(               \
      const void *A, const void *B, void *C, const int32_t *offsets, RockTokenWeightParams p) {       \
    rk::token_weight_body_any<ROCK_DT, BM, BN, WM, WN>(A, B, C, offsets, p);                      \
  }
