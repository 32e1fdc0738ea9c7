// Operators over the token rows of a language model: quantisation row by row, the int8 product with a scale for each
// token and channel, and products whose rows are spread over groups of weights (experts) with their two gradients.
// The reference has no counterpart: its GEMM takes one size for all batch entries (RockOps.td:63-99) and quantises per
// tensor or per channel (MIGraphXToTosa.cpp:874-982).
#include "rock_host.h"

namespace rockhost {

namespace {

struct TokenTile {
  const char *suffix;
  int bm, bn, waves_m, waves_n;
  double cost; // of one tile, the 256 x 256 tile's being 1
};
// Measured with bf16 rows over 8 experts 2048 -> 4096 (us, rows 1024 / 2048 / 4096): 64 x 64 tiles 53 / 72 / 150 with
// 4 / 8 / 16 of them per compute unit, 128 x 128 tiles 47 / 56 / 108 with 1 / 2 / 4, 256 x 256 tiles 49 / 51 / 92.
const TokenTile kTokenTiles[] = {{"_256x256", 256, 256, 2, 4, 1.0}, {"_128x128", 128, 128, 2, 2, 0.47}, {"_64x64", 64, 64, 2, 2, 0.165}};

// The time `tiles` tiles take, in tiles of 256 x 256.  The last of those run in parts (token_gemm.h: tail_parts).
double tile_time(const TokenTile &t, int64_t tiles) {
  if (t.bm < 256)
    return (double)((tiles + kNumCU - 1) / kNumCU) * t.cost;
  const int64_t left = tiles % kNumCU;
  return (double)(tiles / kNumCU) + (left == 0 ? 0.0 : left * 4 <= kNumCU ? 0.4 : left * 2 <= kNumCU ? 0.6 : 1.0);
}

const TokenTile *requested_tile(const OptMap &o) {
  for (const TokenTile &t : kTokenTiles)
    if (requested_tile_is(o, t.bm, t.bn))
      return &t;
  return nullptr;
}

// Kernels for few rows (csrc/token_gemm.h): a block of eight waves per tile, K divided over the waves.
const TokenTile kSkinnyTiles[] = {{"_16x16_skinny", 16, 16, 1, 8, 0.0}, {"_16x32_skinny", 16, 32, 1, 8, 0.0},
                                  {"_32x16_skinny", 32, 16, 1, 8, 0.0}, {"_32x32_skinny", 32, 32, 1, 8, 0.0}};

// The tile for a product of `rows` rows in `groups` groups, or NULL: the tiled kernels.  Measured (i8, times in us in a
// graph): the smallest tile whose blocks leave no compute unit two of them reads the fewest bytes per block, 16 rows of
// 4096 x 4096 9.0 at 16 x 16 against 14.0 on 64 x 64 tiles, 64 rows of 1024 x 4096 7.1 against 13.7; with more blocks
// than units the 64 x 64 tiles with three K-steps in flight stream as fast (16384 x 4096, one row: 19.7 against 19.2)
// and take 64 rows at the same price, so only groups of one or two rows stay here (64 experts 2048 x 4096 at 64 rows: 71
// against 79; at 256 rows 120 against 117).  `aligned`: the tiled kernels' 16-byte chunks fit; if not, the alternative
// is the register-staged kernel, which is slower (f16, 20 experts 1001 x 515 at 51 rows each: 15 against 27 here).
const TokenTile *pick_skinny_tile(int64_t rows, int64_t groups, int64_t cols, bool aligned, const OptMap &o) {
  for (const TokenTile &t : kSkinnyTiles)
    if (requested_tile_is(o, t.bm, t.bn))
      return &t;
  if (requested_tile(o))
    return nullptr;
  const int64_t used = std::min(rows, groups), per_group = ceil_div(rows, used);
  for (int i : {0, 1, 2, 3})
    if (used * ceil_div(per_group, kSkinnyTiles[i].bm) * ceil_div(cols, kSkinnyTiles[i].bn) <= kNumCU)
      return &kSkinnyTiles[i];
  if (per_group <= (aligned ? 2 : 16))
    return &kSkinnyTiles[1];
  return nullptr;
}

// The most row tiles of bm rows that `rows` rows in `groups` groups can make: every group that has a row may end in a
// partial tile.
int64_t row_tiles(int64_t rows, int64_t groups, int64_t bm) {
  const int64_t used = std::min(rows, groups);
  return used ? (rows - used) / bm + used : 0;
}

// Rows spread evenly: what the tile choice expects (how they really lie is known on the device only).
int64_t expected_row_tiles(int64_t rows, int64_t groups, int64_t bm) {
  const int64_t used = std::min(rows, groups);
  return used * ceil_div(ceil_div(rows, used), bm);
}

// The tile with the least time for a product of `rows` rows in `groups` groups with `cols` columns.
const TokenTile *pick_token_tile(int64_t rows, int64_t groups, int64_t cols, const OptMap &o) {
  const TokenTile *best = requested_tile(o);
  double best_time = 0;
  if (best)
    return best;
  for (const TokenTile &t : kTokenTiles) {
    const double time = tile_time(t, expected_row_tiles(rows, groups, t.bm) * ceil_div(cols, t.bn));
    if (!best || time < best_time) {
      best = &t;
      best_time = time;
    }
  }
  return best;
}

// The tile of a weight gradient: `groups` results of M x N, each the sum over about `depth` rows.  The large tile pays
// where the reduction is long (8 experts 4096 x 2048 bf16, us: 2048 rows each 242 against 294 on 128 x 128 and 566 on
// 64 x 64; 256 rows 60 / 58 / 85), short ones are bound by their results and the latency of each tile, which the three
// resident blocks of the 128 x 128 kernel hide (60 experts 1408 x 2048 at 83 rows 98 / 92 / 139; 64 experts 768 x 1024 at
// 16 rows 30 / 23 / 33); few tiles want to be small (4 experts 512 x 512 at 1000 rows 15 / 18 / 14).  f32 results
// stage in twice the LDS and the 128 x 128 kernel has two blocks (8 experts 1024 x 1024 at 250 rows 60 / 49 / 45).
const TokenTile *pick_weight_tile(int64_t groups, int64_t M, int64_t N, int64_t depth, int es, const OptMap &o) {
  if (const TokenTile *t = requested_tile(o))
    return t;
  auto tiles = [&](const TokenTile &t) { return groups * ceil_div(M, t.bm) * ceil_div(N, t.bn); };
  if (depth >= 512 && tiles(kTokenTiles[0]) >= kNumCU / 2)
    return &kTokenTiles[0];
  return &kTokenTiles[tiles(kTokenTiles[1]) >= (es == 4 ? 4 : 1) * kNumCU ? 1 : 2];
}

// Operands of any alignment: 128 x 128 where `tiles` such tiles fill the chip twice (int8 4000 x 4096 x 2051: 94 us
// against 129), else 64 x 64 (1001 x 2307 x 1283: 19 either way; 20 f16 experts 1001 x 515 at 51 rows 13 against 17).
const TokenTile *pick_any_tile(int64_t tiles, const OptMap &o) {
  const TokenTile *t = requested_tile(o);
  return t && t->bm <= 128 ? t : &kTokenTiles[tiles >= 2 * kNumCU ? 1 : 2];
}

std::string token_perf_string(int bm, int bn, int waves_m, int es) {
  char buf[96];
  std::snprintf(buf, sizeof buf, "v2:%d,%d,8,%d,16,%d,1,1,1", bm, bn, bm / waves_m, 16 / es);
  return buf;
}

struct TokenProblem {
  int t, out; // operand and result type
  int64_t G, T, N, K;
  bool transB, token_scale, channel_scale;
};

bool parse_token_problem(const OptMap &o, const char *what, bool grouped, TokenProblem &q) {
  auto fail = [&](const std::string &why) {
    set_error(std::string(what) + ": " + why);
    return false;
  };
  q.t = parse_dtype(str_or(o, "t", "f32"));
  if (q.t != ROCK_F32 && q.t != ROCK_F16 && q.t != ROCK_BF16 && q.t != ROCK_I8)
    return fail("operands are f32, f16, bf16 or i8");
  q.G = int_or(o, "g", 1);
  if (!get_int(o, "m", q.T) || !get_int(o, "n", q.N) || !get_int(o, "k", q.K) || q.G <= 0 || q.T <= 0 || q.N <= 0 ||
      q.K <= 0 || q.T > INT32_MAX - 512 || q.N > INT32_MAX - 512 || q.K > INT32_MAX - 512 || q.G > 65536)
    return fail("-m, -n, -k (and -g) must be given, positive and within 31 bits (-g: at most 65536, every block reads the offsets)");
  q.transB = bool_or(o, "transB", false);
  if (bool_or(o, "transA", false) || bool_or(o, "transC", false))
    return fail("the token rows of operand and result are contiguous (no transA, transC)");
  q.token_scale = bool_or(o, "token_scale_vector", false);
  q.channel_scale = bool_or(o, "scale_vector", false);
  const std::string outs = str_or(o, "out_datatype", "");
  q.out = outs.empty() ? (q.t == ROCK_I8 ? ROCK_F16 : q.t) : parse_dtype(outs);
  if (q.out != ROCK_F32 && q.out != ROCK_F16 && q.out != ROCK_BF16)
    return fail("the result is f32, f16 or bf16");
  if (q.t != ROCK_I8 && (q.token_scale || q.channel_scale || o.count("scale")))
    return fail("scales go with int8 operands");
  if (q.t == ROCK_I8 && q.K > 131071)
    return fail("a reduction of more than 131071 int8 products does not fit the 32-bit sums");
  // what the epilogue of these kernels has no step for
  for (const char *key : {"zero_point_vector", "quant_scale_vector", "out_zero_point_vector", "residual", "quant_scale",
                          "out_zero_point"})
    if (o.count(key) && str_or(o, key, "") != "false" && str_or(o, key, "") != "none")
      return fail(std::string("no ") + key + " beside token rows");
  if (grouped)
    for (const char *key : {"bias", "relu", "activation", "zero_point"})
      if (o.count(key) && str_or(o, key, "") != "false" && str_or(o, key, "") != "none" && str_or(o, key, "") != "0")
        return fail(std::string("no ") + key + " in a product grouped by expert");
  if (int_or(o, "kernel_id", 0) != 0)
    return fail("kernel_id out of range");
  return true;
}

std::string token_key(const OptMap &o, const Handle *h, const TokenProblem &q, const std::string &op) {
  std::ostringstream k;
  k << h->arch << '\t' << int_or(o, "num_cu", kNumCU) << '\t' << (op == "gemm" ? "" : "-operation " + op + " ") << "-t "
    << dtype_name(q.t) << " -out_datatype " << dtype_name(q.out) << " -transA false -transB " << (q.transB ? "true" : "false")
    << " -g " << q.G << " -m " << q.T << " -n " << q.N << " -k " << q.K;
  if (q.token_scale)
    k << " -token_scale_vector true";
  return k.str();
}

bool set_grid(Handle *h, int64_t blocks, int threads, const char *what) {
  if (blocks <= 0 || blocks > INT32_MAX || blocks * threads > 0xffffffffll) {
    set_error(std::string(what) + ": more tiles than one launch can hold");
    return false;
  }
  h->grid_size = (uint32_t)blocks;
  h->block_size = (uint32_t)threads;
  return true;
}

// A product of T rows with `cols` columns over `depth`: b stored [cols, depth] (b_rows) or [depth, cols], groups b_gs
// elements apart.  The kernel's pointers: rows, weights, result, bias, offsets, token scales, channel scales.
bool plan_token_gemm(Handle *h, const TokenProblem &q, int64_t cols, int64_t depth, bool b_rows, const OptMap &o,
                     const char *what) {
  auto &p = reinterpret_cast<RockTokenGemmParams *>(h->params.data())->gemm;
  const int es = dtype_size(q.t);
  p.G = (int)q.G; p.M = (int)q.T; p.N = (int)cols; p.K = (int)depth;
  p.a_ms = depth; p.a_ks = 1;
  p.b_gs = cols * depth; p.b_ns = b_rows ? depth : 1; p.b_ks = b_rows ? 1 : cols;
  p.c_ms = cols; p.c_ns = 1;
  // vector path: rows of whole 16-byte chunks, byte offsets inside a tile below 2^31 (plan_gemm.cpp)
  const int64_t kMaxOff = (int64_t)1 << 31;
  auto al16 = [&](int64_t elems) { return (elems * es) % 16 == 0; };
  const bool a_ok = al16(depth) && 257 * depth * es < kMaxOff;
  const bool b_ok = b_rows ? a_ok : al16(cols) && depth * cols * es + 256 * es < kMaxOff;
  const std::string name = std::string("rock_token_gemm_") + dtype_name(q.t);
  int64_t tiles_m;
  if (const TokenTile *t = b_rows ? pick_skinny_tile(q.T, q.G, cols, a_ok, o) : nullptr) {
    tiles_m = row_tiles(q.T, q.G, t->bm);
    p.tiles_n = ceil_div(cols, t->bn);
    p.group_m = 8;
    h->kernel_name = name + t->suffix;
    h->perf_config = token_perf_string(t->bm, t->bn, 1, es);
    if (!set_grid(h, tiles_m * p.tiles_n, 512, what))
      return false;
  } else if (a_ok && b_ok) {
    const TokenTile *t = pick_token_tile(q.T, q.G, cols, o);
    tiles_m = row_tiles(q.T, q.G, t->bm);
    p.tiles_n = ceil_div(cols, t->bn);
    p.group_m = t->bm >= 256 ? 4 : 8;
    h->kernel_name = name + t->suffix + "_fast" + (b_rows ? "" : "_nn");
    h->perf_config = token_perf_string(t->bm, t->bn, t->waves_m, es);
    // (the last tiles of the largest kernel are cut into parts: up to one block per unit more, kUnits of token_gemm.h)
    if (!set_grid(h, tiles_m * p.tiles_n + (t->bm == 256 ? kNumCU : 0), t->waves_m * t->waves_n * 64, what))
      return false;
  } else {
    const TokenTile *t = pick_any_tile(expected_row_tiles(q.T, q.G, 128) * ceil_div(cols, 128), o);
    tiles_m = row_tiles(q.T, q.G, t->bm);
    p.tiles_n = ceil_div(cols, t->bn);
    p.group_m = 8;
    h->kernel_name = name + t->suffix + "_any" + (b_rows ? "" : "_nn");
    h->perf_config = token_perf_string(t->bm, t->bn, t->waves_m, es);
    if (!set_grid(h, tiles_m * p.tiles_n, 256, what))
      return false;
  }
  p.tiles_m = (int)tiles_m;
  p.group_m = std::min(p.group_m, p.tiles_m);
  p.xcd_remap = h->grid_size >= 2 * kNumXCD ? 1 : 0;
  h->num_pointers = 7;
  return true;
}

} // namespace

// C = (A B - zero_point) * scale[n] * token_scale[m] + bias: caller list A, B, C, bias, token scales, [channel scales]
Handle *make_token_scaled_gemm(const OptMap &o) {
  TokenProblem q;
  if (!parse_token_problem(o, "gemm with token scales", false, q))
    return nullptr;
  if (q.t != ROCK_I8 || q.G != 1) {
    set_error("gemm with token scales: int8 operands, one batch entry");
    return nullptr;
  }
  auto *h = new Handle;
  h->op = OP_GEMM;
  h->params.assign(sizeof(RockTokenGemmParams), 0);
  auto &p = reinterpret_cast<RockTokenGemmParams *>(h->params.data())->gemm;
  h->epi = &p.epi;
  OptMap scalars = o; // (the channel scales are a pointer of these kernels, not of the epilogue block)
  scalars.erase("scale_vector");
  if (!parse_epilogue(scalars, q.t, q.out, p.epi) || p.epi.activation > ROCK_ACT_CLIP) {
    set_error("gemm with token scales: scale, zero_point, bias and the activations relu and clip");
    delete h;
    return nullptr;
  }
  if (!plan_token_gemm(h, q, q.N, q.K, q.transB, o, "gemm with token scales")) {
    delete h;
    return nullptr;
  }
  h->ptr_map = {{0, 0}, {1, 0}, {2, 0}, {3, 0}, {-1, 0}, {4, 0}, {q.channel_scale ? 5 : -1, 0}};
  h->caller_pointers = q.channel_scale ? 6 : 5;
  h->problem_key = token_key(o, h, q, "gemm");
  h->args = {{q.t, {1, q.T, q.K}}, {q.t, q.transB ? std::vector<int64_t>{1, q.N, q.K} : std::vector<int64_t>{1, q.K, q.N}},
             {q.out, {1, q.T, q.N}}, {ROCK_F32, {q.N}}, {ROCK_F32, {q.T}}};
  if (q.channel_scale)
    h->args.push_back({ROCK_F32, {q.N}});
  return h;
}

// Products grouped by expert.  Every direction takes the forward problem's keys and pointer order -- rows, weights,
// result, offsets, [token scales,] [channel scales] -- and a gradient is written in its own slot, as for the
// convolutions (rocmlir-lib.cpp:150-199).
Handle *make_grouped_gemm(const OptMap &o) {
  const std::string op = str_or(o, "operation", "");
  TokenProblem q;
  if (!parse_token_problem(o, op.c_str(), true, q))
    return nullptr;
  const bool forward = op == "grouped_gemm", weight = op == "grouped_gemm_bwd_weight";
  if (!forward && q.t == ROCK_I8) {
    set_error(op + ": gradients take f32, f16 or bf16");
    return nullptr;
  }
  if (!forward && q.out != q.t) {
    set_error(op + ": a gradient has its tensor's type");
    return nullptr;
  }
  auto *h = new Handle;
  h->op = OP_TOKENS;
  h->args = {{q.t, {q.T, q.K}}, {q.t, q.transB ? std::vector<int64_t>{q.G, q.N, q.K} : std::vector<int64_t>{q.G, q.K, q.N}},
             {q.out, {q.T, q.N}}, {ROCK_I32, {q.G + 1}}};
  h->problem_key = token_key(o, h, q, op);
  h->caller_pointers = 4;
  if (weight) {
    h->params.assign(sizeof(RockTokenWeightParams), 0);
    auto &p = reinterpret_cast<RockTokenWeightParams *>(h->params.data())->gemm;
    default_epilogue(p.epi, q.out);
    // stored [N, K]: rows of the result run over the forward result's columns; stored [K, N]: over the rows' columns
    const int64_t M = q.transB ? q.N : q.K, N = q.transB ? q.K : q.N;
    const int es = dtype_size(q.t);
    p.G = (int)q.G; p.M = (int)M; p.N = (int)N; p.K = (int)q.T;
    p.a_ms = 1; p.a_ks = M;
    p.b_ns = 1; p.b_ks = N;
    p.c_gs = M * N; p.c_ms = N; p.c_ns = 1;
    const int64_t kMaxOff = (int64_t)1 << 31;
    auto cols_ok = [&](int64_t c) { return (c * es) % 16 == 0 && (128 / es) * c * es + 512 < kMaxOff; };
    const std::string name = std::string("rock_token_gemm_bwd_weight_") + dtype_name(q.t);
    int bm = 64, bn = 64, threads = 256;
    if (cols_ok(M) && cols_ok(N)) {
      const TokenTile *t = pick_weight_tile(q.G, M, N, ceil_div(q.T, std::min(q.T, q.G)), es, o);
      bm = t->bm; bn = t->bn;
      threads = t->waves_m * t->waves_n * 64;
      h->kernel_name = name + t->suffix;
      h->perf_config = token_perf_string(bm, bn, t->waves_m, es);
      // the reduction over the waves of a block: where the 64 x 64 tiles leave no compute unit two of them and every
      // share has two K-steps (bf16, us with / without: one result 512 x 512 of 4000 rows 23 / 34, 256 x 256 of 16384 75 /
      // 126, four 512 x 512 of 1000 rows each 11 / 13, of 250 6.6 / 5.2); splitK, the seventh field of a perf_config,
      // asks for it or declines it
      const int64_t tiles = q.G * ceil_div(M, 64) * ceil_div(N, 64), depth = ceil_div(q.T, std::min(q.T, q.G));
      const bool asked = o.count("perf_config") && bm == 64 && requested_tile(o);
      if (bm == 64 && (asked ? perf_field(o, 6, 1) == 4 : tiles <= kNumCU && depth * es >= 8 * 128)) {
        threads = 1024;
        h->kernel_name = name + "_64x64_split";
        h->perf_config = with_block_splits(h->perf_config, 4);
      }
    } else {
      const TokenTile *t = pick_any_tile(q.G * ceil_div(M, 128) * ceil_div(N, 128), o);
      bm = t->bm; bn = t->bn;
      h->kernel_name = name + t->suffix + "_any";
      h->perf_config = token_perf_string(bm, bn, t->waves_m, es);
    }
    p.tiles_m = ceil_div(M, bm);
    p.tiles_n = ceil_div(N, bn);
    p.group_m = std::min(p.tiles_m, bm >= 256 ? 4 : 8);
    int64_t blocks = q.G * p.tiles_m * (int64_t)p.tiles_n;
    if (blocks > INT32_MAX)
      blocks = -1;
    else if (bm == 256)
      blocks += kNumCU; // the last tiles in parts, as above
    if (!set_grid(h, blocks, threads, op.c_str())) {
      delete h;
      return nullptr;
    }
    h->num_pointers = 4;
    h->ptr_map = {{q.transB ? 2 : 0, 0}, {q.transB ? 0 : 2, 0}, {1, 0}, {3, 0}};
    return h;
  }
  h->params.assign(sizeof(RockTokenGemmParams), 0);
  auto &p = reinterpret_cast<RockTokenGemmParams *>(h->params.data())->gemm;
  default_epilogue(p.epi, q.out);
  if (forward && q.t == ROCK_I8) {
    get_float(o, "scale", p.epi.scale);
    h->epi = &p.epi;
  }
  const bool ok = forward ? plan_token_gemm(h, q, q.N, q.K, q.transB, o, op.c_str())
                          : plan_token_gemm(h, q, q.K, q.N, !q.transB, o, op.c_str());
  if (!ok) {
    delete h;
    return nullptr;
  }
  int next = 4;
  const int token = q.token_scale ? next++ : -1, channel = q.channel_scale ? next++ : -1;
  if (q.token_scale)
    h->args.push_back({ROCK_F32, {q.T}});
  if (q.channel_scale)
    h->args.push_back({ROCK_F32, {q.G, q.N}});
  h->caller_pointers = next;
  h->ptr_map = {{forward ? 0 : 2, 0}, {1, 0}, {forward ? 2 : 0, 0}, {-1, 0}, {3, 0}, {token, 0}, {channel, 0}};
  return h;
}

// Rows to int8 with a scale each: caller list x [m, k], q [m, k], scales [m]
Handle *make_quantize_tokens(const OptMap &o) {
  const int t = parse_dtype(str_or(o, "t", "f16"));
  int64_t rows, cols;
  if ((t != ROCK_F32 && t != ROCK_F16 && t != ROCK_BF16) || !get_int(o, "m", rows) || !get_int(o, "k", cols) ||
      rows <= 0 || cols <= 0 || cols > INT32_MAX - 512 || rows > INT32_MAX - 512) {
    set_error("quantize_tokens: -t f32|f16|bf16, -m rows and -k columns, positive and within 31 bits");
    return nullptr;
  }
  if (int_or(o, "kernel_id", 0) != 0) {
    set_error("quantize_tokens: kernel_id out of range");
    return nullptr;
  }
  auto *h = new Handle;
  h->op = OP_TOKENS;
  h->params.assign(sizeof(RockQuantizeParams), 0);
  auto &p = *reinterpret_cast<RockQuantizeParams *>(h->params.data());
  p.rows = rows;
  p.cols = (int32_t)cols;
  // a wave holds rows of up to 8 KiB in registers; few rows take the whole block each so that more lanes load
  p.lanes_per_row = cols * dtype_size(t) > 8192 || rows < 1024 ? 256 : 64;
  h->kernel_name = std::string("rock_quantize_tokens_") + dtype_name(t);
  if (!set_grid(h, p.lanes_per_row == 64 ? (rows + 3) / 4 : rows, 256, "quantize_tokens")) {
    delete h;
    return nullptr;
  }
  h->num_pointers = 3;
  std::ostringstream key;
  key << h->arch << '\t' << int_or(o, "num_cu", kNumCU) << "\t-operation quantize_tokens -t " << dtype_name(t) << " -m " << rows
      << " -k " << cols;
  h->problem_key = key.str();
  h->args = {{t, {rows, cols}}, {ROCK_I8, {rows, cols}}, {ROCK_F32, {rows}}};
  return h;
}

} // namespace rockhost
