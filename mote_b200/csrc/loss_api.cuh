// C-ABI entry points of the losses on logits (include/moteopt.h): argument checks, the choice of kernels and the launches.
// Included by moteopt.cu, whose error and launch macros it uses. No device memory is allocated here, nothing synchronises.
#pragma once

namespace {

using namespace moteopt::loss;

// Rows of up to this many bytes take tile_kernel, a warp for several rows; longer ones a block or more each.
constexpr int64_t kShortBytes = kTileBytes - 32;

constexpr int64_t kSliceBytes = 72 * 1024, kSliceMost = 220 * 1024, kSliceLeast = 8 * 1024;
constexpr int64_t kRowMost = kMaxCluster * (kSliceMost - 64);   // bytes of the longest row

int64_t esize(int dtype) { return dtype == MOTEOPT_DTYPE_BF16 ? 2 : 4; }

bool positions_fit(const moteopt_logits* z) {
  return z->tokens == 0 || z->seqs <= ((int64_t{1} << 27) - 1) / z->tokens;
}

bool shape_fits(const moteopt_logits* z) {   // for the workspace sizes
  return z && z->seqs >= 0 && z->tokens >= 0 && z->vocab >= 1 &&
         (z->dtype == MOTEOPT_DTYPE_F32 || z->dtype == MOTEOPT_DTYPE_BF16) && z->vocab <= kRowMost / esize(z->dtype) &&
         positions_fit(z);
}

int check_logits(const char* who, const moteopt_logits* z, const moteopt_positions* y, Rows* R, double temperature) {
  const std::string w(who);
  if (!z || !y) return fail(MOTEOPT_ERR_INVALID, w + ": null logits or targets");
  if (z->dtype != MOTEOPT_DTYPE_F32 && z->dtype != MOTEOPT_DTYPE_BF16)
    return fail(MOTEOPT_ERR_INVALID, w + ": logits must be fp32 or bf16");
  if (z->seqs < 0 || z->tokens < 0 || z->vocab < 1) return fail(MOTEOPT_ERR_INVALID, w + ": bad logits shape");
  if (z->vocab > kRowMost / esize(z->dtype))
    return fail(MOTEOPT_ERR_LIMIT, w + ": a row of logits may take " + std::to_string(kRowMost) + " bytes");
  if (!positions_fit(z)) return fail(MOTEOPT_ERR_LIMIT, w + ": 2^27 positions or more");
  if (!(static_cast<float>(temperature) > 0.f) || !std::isfinite(static_cast<float>(temperature)) ||
      !std::isfinite(1.f / static_cast<float>(temperature)))
    return fail(MOTEOPT_ERR_INVALID, w + ": the temperature must be positive and finite");
  const int64_t n = z->seqs * z->tokens;
  if (n > 0 && (!z->data || !y->data)) return fail(MOTEOPT_ERR_INVALID, w + ": null logits or targets");
  if (reinterpret_cast<uint64_t>(z->data) % esize(z->dtype) != 0 || reinterpret_cast<uint64_t>(y->data) % 8 != 0)
    return fail(MOTEOPT_ERR_INVALID, w + ": logits or targets are not aligned to their elements");
  std::memset(R, 0, sizeof(*R));
  R->z = static_cast<const char*>(z->data);
  R->y = static_cast<const int64_t*>(y->data);
  R->z_seq = z->seq_stride;
  R->z_tok = z->token_stride;
  R->y_seq = y->seq_stride;
  R->y_tok = y->token_stride;
  R->n = static_cast<uint32_t>(n);
  R->tokens = static_cast<uint32_t>(z->tokens);
  R->vocab = static_cast<uint32_t>(z->vocab);
  // as torch divides fp32 by a number: a product with its fp32 reciprocal. Old log-probabilities that a sampler formed that way
  // are of the same x (with the exact 1 / T the mean logp at T = 0.9 and 131072 logits is 1.7e-7 away).
  R->inv_t = static_cast<double>(1.f / static_cast<float>(temperature));
  R->t = 1.0 / R->inv_t;
  const double c = kLog2e * R->inv_t;
  int exp = 0;
  double bits = std::floor(std::ldexp(std::frexp(c, &exp), 12));   // c_hi: 12 bits, below c
  if (std::ldexp(bits, exp - 12) >= c) bits -= 1.0;
  const float hi = static_cast<float>(std::ldexp(bits, exp - 12));
  R->c_hi = hi;
  R->c_lo = static_cast<float>(c - static_cast<double>(hi));
  if (!(R->c_lo >= FLT_MIN) || !std::isfinite(hi)) return fail(MOTEOPT_ERR_INVALID, w + ": the temperature is out of range");
  return MOTEOPT_OK;
}

// Pointers of a call, each aligned to its elements of `size` bytes (null ones are)
int check_aligned(const char* who, size_t size, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uint64_t>(p) % size != 0)
      return fail(MOTEOPT_ERR_INVALID, std::string(who) + ": a tensor is not aligned to its elements");
  return MOTEOPT_OK;
}

Per per_of(const moteopt_positions& p) { return Per{static_cast<const float*>(p.data), p.seq_stride, p.token_stride}; }

// A launch behind another one of the same call: its blocks may be placed before that one has ended (they wait for it
// themselves). The first launch of a call (`first`) is an ordinary one.
template <typename Args>
int launch_after(void (*kernel)(Args), const Args& A, unsigned grid, unsigned block, size_t smem, cudaStream_t st,
                 const char* what, bool first = false) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = first ? 0 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A);
  if (e != cudaSuccess) return fail(MOTEOPT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return MOTEOPT_OK;
}

template <typename Args>
int launch_cluster(void (*kernel)(Args), const Args& A, unsigned rows, unsigned cl, unsigned block, size_t smem,
                   cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * cl, 1, 1);
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cl > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A);
  if (e != cudaSuccess) return fail(MOTEOPT_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return MOTEOPT_OK;
}

bool short_rows(int dtype, int64_t vocab) { return vocab * esize(dtype) <= kShortBytes; }

// Tiles: as many rows as fit kTileBytes, at most kTileRows, and fewer while that would leave an SM less than 24 warps (a warp
// takes its rows four at a time, one lot after the other). Lanes per row: 8, and the whole warp where a row has more than 16
// lines for each of them.
constexpr uint32_t kNarrowPitch = 8 * 16 * 16;
struct TileShape {
  int per_warp;
  uint32_t pitch, tiles;
};
TileShape tile_shape(int64_t rows, int64_t line_bytes, int sms) {
  TileShape s;
  s.pitch = static_cast<uint32_t>((line_bytes / 16 + 1) * 16);
  const int64_t most = std::min<int64_t>(kTileRows, kTileBytes / s.pitch);
  s.per_warp = static_cast<int>(std::max<int64_t>(1, std::min(most, rows / (24 * sms))));
  s.tiles = static_cast<uint32_t>(cdiv(rows, s.per_warp));
  return s;
}
int64_t line_bytes(int dtype, int64_t vocab) { return (vocab * esize(dtype) + 16 - esize(dtype) + 15) / 16 * 16; }

// 8 lanes a row with at most 2 or 5 lines each, or more, or 32 lanes a row. (10 lines each take so many registers that 8 x 2048
// x 271 fp32, forward, takes 7.1 us and not 6.1.)
template <typename T, Mode kMode>
auto tile_fn(uint32_t pitch) {
  const uint32_t lines = pitch / 16 - 1;
  return pitch > kNarrowPitch ? tile_kernel<T, 32, 0, kMode>
         : lines <= 16        ? tile_kernel<T, 8, 2, kMode>
         : lines <= 40        ? tile_kernel<T, 8, 5, kMode>
                              : tile_kernel<T, 8, 0, kMode>;
}
template <Mode kMode>
auto tile_fn(int dtype, uint32_t pitch) {
  return dtype == MOTEOPT_DTYPE_BF16 ? tile_fn<__nv_bfloat16, kMode>(pitch) : tile_fn<float, kMode>(pitch);
}
size_t tile_smem(const TileShape& s) { return static_cast<size_t>(kTileWarps) * s.per_warp * s.pitch; }

template <Mode kMode>
int launch_tile(int dtype, TileArgs A, const TileShape& s, cudaStream_t st, bool after = false) {
  A.per_warp = s.per_warp;
  A.pitch = s.pitch;
  return launch_after(tile_fn<kMode>(dtype, s.pitch), A, static_cast<unsigned>(cdiv(s.tiles, kTileWarps)), kTileWarps * 32,
                      tile_smem(s), st, "loss tile_kernel", !after);
}
// Few rows: the policy or the preference loss in one launch of one cluster, whose blocks' sums meet in its first block, or whose
// blocks share out the pairs. Two lots of rows a warp take no longer than the launches that this saves.
bool one_cluster(int64_t rows, const TileShape& s) {
  return rows <= static_cast<int64_t>(kMaxCluster) * kTileWarps * (s.pitch <= kNarrowPitch ? 8 : 1) &&
         (s.pitch > kNarrowPitch || 8 * s.pitch <= kTileBytes);
}
constexpr int kClusterPairs = 256;
template <Mode kMode>
int launch_tile_cluster(int dtype, TileArgs A, TileShape s, cudaStream_t st) {
  unsigned blocks = 1;
  while (blocks < kMaxCluster && static_cast<int64_t>(blocks) * kTileWarps < A.R.n) blocks *= 2;
  s.per_warp = static_cast<int>(cdiv(A.R.n, blocks * kTileWarps));
  A.per_warp = s.per_warp;
  A.pitch = s.pitch;
  return launch_cluster(tile_fn<kMode>(dtype, s.pitch), A, 1, blocks, kTileWarps * 32, tile_smem(s), st,
                        "loss tile_kernel");
}

// Long rows: blocks per row and bytes of shared memory each. A slice of up to kSliceBytes leaves three blocks an SM; a
// row that 16 such slices do not hold takes larger ones, one block an SM. Where there are too few rows for the
// GPU they are cut further, down to kSliceLeast.
struct SliceShape {
  int threads, cl;
  size_t smem;
};
SliceShape slice_shape(int64_t rows, int64_t vocab, int dtype, int sms) {
  const int64_t bytes = vocab * esize(dtype);
  SliceShape s = {256, 1, 0};
  const auto smem = [&](int cl) { return (cdiv(bytes / 16, cl) + 4) * 16; };   // 3 lines beside the share, 1 to read over
  while (s.cl < kMaxCluster && smem(s.cl) > kSliceBytes) s.cl *= 2;
  while (s.cl < kMaxCluster && rows * s.cl * 2 <= 2 * sms && smem(s.cl * 2) >= kSliceLeast) s.cl *= 2;
  s.smem = static_cast<size_t>(smem(s.cl));
  if (s.smem <= kSliceBytes / 4) s.threads = 128;
  return s;
}

int launch_slices(int dtype, SliceArgs A, int sms, cudaStream_t st) {
  const SliceShape s = slice_shape(A.R.n, A.R.vocab, dtype, sms);
  const bool bf = dtype == MOTEOPT_DTYPE_BF16;
  A.cl = s.cl;
  auto* const k = s.threads == 128 ? (bf ? slice_kernel<__nv_bfloat16, 128> : slice_kernel<float, 128>)
                                   : (bf ? slice_kernel<__nv_bfloat16, 256> : slice_kernel<float, 256>);
  return launch_cluster(k, A, A.R.n, s.cl, s.threads, s.smem, st, "loss slice_kernel");
}

// Long rows go in pieces, whose parts are kept: pieces of a row, and the bytes of all parts. Pieces of 256, 512 and 1024 lines:
// 4 x 2048 x 8192 bf16 36.4, 34.4 and 32.8 us, 8 rows of 262144 fp32 8.8, 7.2 and 6.7 us. Four times the blocks that fit an SM,
// so that one that falls behind takes fewer: 4 x 1024 x 32768, 52.4 against 51.1 us.
constexpr uint32_t kPieceLines = 1024;
constexpr int kStreamGrid = 4 * 8;   // blocks per SM in all
// A row's lines are shared out in whole batches, in the number of pieces of 5/8 to 5/4 of kPieceLines that leaves the last one
// the least short.
struct PieceShape {
  int64_t pieces, lines;
};
PieceShape piece_shape(int dtype, int64_t vocab) {
  constexpr int64_t kBatchLines = 32 * kBatch;
  const int64_t all = line_bytes(dtype, vocab) / 16;
  const int64_t least = std::max<int64_t>(1, cdiv(all * 4, kPieceLines * 5)), most = std::max(least, all * 8 / (kPieceLines * 5));
  PieceShape best = {0, 0};
  for (int64_t p = least; p <= most; ++p) {
    const int64_t lines = cdiv(cdiv(all, p), kBatchLines) * kBatchLines;
    if (best.pieces == 0 || p * lines < best.pieces * best.lines) best = {p, lines};
  }
  return best;
}
int64_t row_pieces(int dtype, int64_t vocab) { return piece_shape(dtype, vocab).pieces; }
size_t parts_bytes(int dtype, int64_t rows, int64_t vocab) {
  return short_rows(dtype, vocab) ? 0 : sizeof(Part) * static_cast<size_t>(rows) * static_cast<size_t>(row_pieces(dtype, vocab));
}

// logp, lse (or logp64, lse64, coef = 0) of every row
int launch_forward(int dtype, const Rows& R, float* logp, float* lse, double* logp64, double* lse64, float* coef, Part* parts,
                   int sms, cudaStream_t st) {
  if (short_rows(dtype, R.vocab)) {
    TileArgs A;
    std::memset(&A, 0, sizeof(A));
    A.R = R;
    A.logp = logp;
    A.lse = lse;
    A.logp64 = logp64;
    A.lse64 = lse64;
    A.coef = coef;
    return launch_tile<kForward>(dtype, A, tile_shape(R.n, line_bytes(dtype, R.vocab), sms), st);
  }
  const int64_t pieces = row_pieces(dtype, R.vocab);
  if (R.n * pieces >= (int64_t{1} << 31)) return fail(MOTEOPT_ERR_LIMIT, "losses: too many logits for one call");
  StreamArgs A;
  std::memset(&A, 0, sizeof(A));
  A.R = R;
  A.pieces = static_cast<uint32_t>(pieces);
  A.n = R.n * A.pieces;
  A.lines = static_cast<uint32_t>(piece_shape(dtype, R.vocab).lines);
  A.parts = parts;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(cdiv(A.n, kStreamThreads / 32), kStreamGrid * sms));
  MO_TRY(dtype == MOTEOPT_DTYPE_BF16
             ? launch_after(stream_kernel<__nv_bfloat16>, A, blocks, kStreamThreads, kStreamSmem, st, "loss stream_kernel", true)
             : launch_after(stream_kernel<float>, A, blocks, kStreamThreads, kStreamSmem, st, "loss stream_kernel", true));
  JoinArgs J;
  std::memset(&J, 0, sizeof(J));
  J.R = R;
  J.pieces = A.pieces;
  J.parts = parts;
  J.logp = logp;
  J.lse = lse;
  J.logp64 = logp64;
  J.lse64 = lse64;
  J.coef = coef;
  const unsigned grid = static_cast<unsigned>(cdiv(R.n, kJoinThreads / 32));
  return dtype == MOTEOPT_DTYPE_BF16 ? launch_after(join_kernel<__nv_bfloat16>, J, grid, kJoinThreads, 0, st, "loss join_kernel")
                                     : launch_after(join_kernel<float>, J, grid, kJoinThreads, 0, st, "loss join_kernel");
}

int launch_gradient(int dtype, const Rows& R, const Kept& K, void* grad, int sms, cudaStream_t st, bool after) {
  if (short_rows(dtype, R.vocab)) {
    TileArgs A;
    std::memset(&A, 0, sizeof(A));
    A.R = R;
    A.K = K;
    A.grad = grad;
    return launch_tile<kGradient>(dtype, A, tile_shape(R.n, line_bytes(dtype, R.vocab), sms), st, after);
  }
  GradArgs A;
  std::memset(&A, 0, sizeof(A));
  A.R = R;
  A.K = K;
  A.grad = grad;
  A.pieces = static_cast<uint32_t>(cdiv(R.vocab * esize(dtype) / 16, kGradThreads * kGradVecs));
  if (static_cast<int64_t>(R.n) * A.pieces >= (int64_t{1} << 31))
    return fail(MOTEOPT_ERR_LIMIT, "loss gradient: too many logits for one call");
  const unsigned grid = R.n * A.pieces;
  return dtype == MOTEOPT_DTYPE_BF16
             ? launch_after(grad_kernel<__nv_bfloat16>, A, grid, kGradThreads, 0, st, "loss grad_kernel", !after)
             : launch_after(grad_kernel<float>, A, grid, kGradThreads, 0, st, "loss grad_kernel", !after);
}

constexpr int kSumShare = 4096;   // partials one block adds up
constexpr int kSumBlocks = 128;

struct PolicyLayout {
  size_t partials, sums, bytes;
};
PolicyLayout policy_layout(int dtype, int64_t n, int64_t vocab) {
  // a row of partials for each block: of long rows one a position, of short ones at most one for a row a warp. Up to 128 KB are
  // not counted out
  const int64_t rows = short_rows(dtype, vocab) ? std::max(cdiv(n, kTileWarps), std::min<int64_t>(n, kSumShare)) : n;
  PolicyLayout L;
  L.partials = kHeaderBytes;
  L.sums = align_up(L.partials + 32 * static_cast<size_t>(rows), 256);
  L.bytes = L.sums + 32 * kSumBlocks;
  return L;
}

int launch_sums(const double* partials, int64_t n, double* mid, float* out, cudaStream_t st) {
  SumArgs A = {partials, static_cast<uint32_t>(n), mid, out};
  if (n > kSumShare) {
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(kSumBlocks, cdiv(n, kSumShare / 4)));
    MO_TRY(launch_after(sum_kernel, A, blocks, kSumThreads, 0, st, "loss sum_kernel"));
    A.partials = mid;
    A.n = blocks;
  }
  return launch_after(sum_kernel, A, 1, kSumThreads, 0, st, "loss sum_kernel");
}

struct PreferenceLayout {
  size_t logp64, lse, coef, pairs, parts, bytes;
};
PreferenceLayout preference_layout(int dtype, int64_t n, int64_t vocab, int64_t pairs) {
  PreferenceLayout L;
  L.logp64 = kHeaderBytes;
  L.lse = align_up(L.logp64 + 8 * static_cast<size_t>(n), 256);
  L.coef = align_up(L.lse + 8 * static_cast<size_t>(n), 256);
  L.pairs = align_up(L.coef + 4 * static_cast<size_t>(n), 256);
  L.parts = align_up(L.pairs + 8 * static_cast<size_t>(pairs), 256);
  L.bytes = align_up(L.parts + parts_bytes(dtype, n, vocab), 256);
  return L;
}

int check_divisor(const char* who, double divisor, const float* divisor_device) {
  if (!divisor_device && (!(divisor != 0.0) || !std::isfinite(divisor)))
    return fail(MOTEOPT_ERR_INVALID, std::string(who) + ": the divisor must be finite and not 0");
  return MOTEOPT_OK;
}

template <typename K>
int allow_smem(K* kernel, int bytes) {
  MO_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  return MOTEOPT_OK;
}
template <typename K>
int allow_wide(K* kernel) {   // clusters of 16 blocks
  MO_CUDA(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  return MOTEOPT_OK;
}
template <typename T>
int kernel_setup() {
  MO_TRY(allow_smem(slice_kernel<T, 128>, static_cast<int>(kSliceMost)));
  MO_TRY(allow_smem(slice_kernel<T, 256>, static_cast<int>(kSliceMost)));
  MO_TRY(allow_wide(slice_kernel<T, 128>));
  MO_TRY(allow_wide(slice_kernel<T, 256>));
  for (uint32_t lines : {16u, 40u, 100u, 500u}) {
    MO_TRY(allow_wide(tile_fn<T, kPolicyLoss>((lines + 1) * 16)));
    MO_TRY(allow_wide(tile_fn<T, kPreference>((lines + 1) * 16)));
  }
  return MOTEOPT_OK;
}

// the slices' shared memory, and clusters of 16 blocks, are beyond the default limits
int loss_setup(int* sms) {
  MO_TRY(device_setup(sms));
  static std::atomic<unsigned long long> ready{0};   // a bit per device
  int dev = 0;
  MO_CUDA(cudaGetDevice(&dev));
  if (ready.load(std::memory_order_acquire) >> dev & 1) return MOTEOPT_OK;
  MO_TRY(kernel_setup<__nv_bfloat16>());
  MO_TRY(kernel_setup<float>());
  ready.fetch_or(1ull << dev, std::memory_order_release);
  return MOTEOPT_OK;
}

}  // namespace

extern "C" {

size_t moteopt_token_logprobs_workspace_size(const moteopt_logits* logits) {
  if (!shape_fits(logits)) return 0;
  return align_up(kHeaderBytes + parts_bytes(logits->dtype, logits->seqs * logits->tokens, logits->vocab), 256);
}

int moteopt_token_logprobs(const moteopt_logits* logits, const moteopt_positions* targets, double temperature,
                           float* logprobs, float* lse, void* workspace, size_t workspace_bytes, moteopt_stream_t stream) {
  Rows R;
  MO_TRY(check_logits("moteopt_token_logprobs", logits, targets, &R, temperature));
  if (R.n == 0) return MOTEOPT_OK;
  if (!logprobs) return fail(MOTEOPT_ERR_INVALID, "moteopt_token_logprobs: null output");
  MO_TRY(check_aligned("moteopt_token_logprobs", 4, {logprobs, lse}));
  Part* parts = nullptr;
  if (!short_rows(logits->dtype, R.vocab)) {
    MO_TRY(check_ws(workspace, workspace_bytes, moteopt_token_logprobs_workspace_size(logits)));
    parts = reinterpret_cast<Part*>(static_cast<char*>(workspace) + kHeaderBytes);
  }
  int sms = 0;
  MO_TRY(loss_setup(&sms));
  return launch_forward(logits->dtype, R, logprobs, lse, nullptr, nullptr, nullptr, parts, sms,
                        reinterpret_cast<cudaStream_t>(stream));
}

int moteopt_token_logprobs_backward(const moteopt_logits* logits, const moteopt_positions* targets, double temperature,
                                    const moteopt_positions* logprobs, const moteopt_positions* lse,
                                    const moteopt_positions* grad_logprobs, void* grad_logits, moteopt_stream_t stream) {
  Rows R;
  MO_TRY(check_logits("moteopt_token_logprobs_backward", logits, targets, &R, temperature));
  if (R.n == 0) return MOTEOPT_OK;
  if (!logprobs || !lse || !grad_logprobs || !logprobs->data || !lse->data || !grad_logprobs->data || !grad_logits)
    return fail(MOTEOPT_ERR_INVALID, "moteopt_token_logprobs_backward: null pointer");
  MO_TRY(check_aligned("moteopt_token_logprobs_backward", 4, {logprobs->data, lse->data, grad_logprobs->data}));
  MO_TRY(check_aligned("moteopt_token_logprobs_backward", esize(logits->dtype), {grad_logits}));
  int sms = 0;
  MO_TRY(loss_setup(&sms));
  Kept K;
  std::memset(&K, 0, sizeof(K));
  K.logp = per_of(*logprobs);
  K.lse = per_of(*lse);
  K.coef = per_of(*grad_logprobs);
  return launch_gradient(logits->dtype, R, K, grad_logits, sms, reinterpret_cast<cudaStream_t>(stream), false);
}

size_t moteopt_policy_loss_workspace_size(const moteopt_logits* logits) {
  if (!shape_fits(logits)) return 0;
  return policy_layout(logits->dtype, logits->seqs * logits->tokens, logits->vocab).bytes;
}

int moteopt_policy_loss(const moteopt_logits* logits, const moteopt_positions* targets, const moteopt_policy* policy,
                        double temperature, float* sums, float* logprobs, void* grad_logits, void* workspace,
                        size_t workspace_bytes, moteopt_stream_t stream) {
  const char* const who = "moteopt_policy_loss";
  Rows R;
  MO_TRY(check_logits(who, logits, targets, &R, temperature));
  if (!policy || !sums) return fail(MOTEOPT_ERR_INVALID, "moteopt_policy_loss: null pointer");
  MO_TRY(check_divisor(who, policy->divisor, policy->divisor_device));
  if (!(policy->clip_low >= 0.0) || !(policy->clip_high >= 0.0) || !std::isfinite(policy->kl_coef))
    return fail(MOTEOPT_ERR_INVALID, "moteopt_policy_loss: the clips must not be negative, the KL coefficient finite");
  if (R.n > 0 && (!logprobs || !policy->advantages.data || !policy->old_logprobs.data))
    return fail(MOTEOPT_ERR_INVALID, "moteopt_policy_loss: null pointer");
  if (policy->kl_coef != 0.0 && R.n > 0 && !policy->ref_logprobs.data)
    return fail(MOTEOPT_ERR_INVALID, "moteopt_policy_loss: a KL coefficient without reference log-probabilities");
  MO_TRY(check_aligned(who, 4, {sums, logprobs, policy->advantages.data, policy->old_logprobs.data, policy->ref_logprobs.data,
                                policy->weights.data, policy->divisor_device}));
  MO_TRY(check_aligned(who, esize(logits->dtype), {grad_logits}));
  const PolicyLayout L = policy_layout(logits->dtype, R.n, R.vocab);
  MO_TRY(check_ws(workspace, workspace_bytes, L.bytes));
  int sms = 0;
  MO_TRY(loss_setup(&sms));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (R.n == 0) {
    MO_CUDA(cudaMemsetAsync(sums, 0, 4 * sizeof(float), st));
    return MOTEOPT_OK;
  }
  char* const ws = static_cast<char*>(workspace);
  Policy P;
  std::memset(&P, 0, sizeof(P));
  P.adv = per_of(policy->advantages);
  P.old_lp = per_of(policy->old_logprobs);
  P.ref_lp = per_of(policy->ref_logprobs);
  P.weight = per_of(policy->weights);
  P.clip_lo = 1.0 - policy->clip_low;
  P.clip_hi = 1.0 + policy->clip_high;
  P.kl = policy->kl_coef;
  P.inv_div = policy->divisor_device ? 0.0 : 1.0 / policy->divisor;
  P.div = policy->divisor_device;
  double* const partials = reinterpret_cast<double*>(ws + L.partials);
  double* const mid = reinterpret_cast<double*>(ws + L.sums);
  if (short_rows(logits->dtype, R.vocab)) {
    TileArgs A;
    std::memset(&A, 0, sizeof(A));
    A.R = R;
    A.P = P;
    A.logp = logprobs;
    A.grad = grad_logits;
    A.partials = partials;
    const TileShape s = tile_shape(R.n, line_bytes(logits->dtype, R.vocab), sms);
    if (one_cluster(R.n, s)) {
      A.sums = sums;
      return launch_tile_cluster<kPolicyLoss>(logits->dtype, A, s, st);
    }
    MO_TRY(launch_tile<kPolicyLoss>(logits->dtype, A, s, st));
    return launch_sums(partials, cdiv(s.tiles, kTileWarps), mid, sums, st);
  }
  SliceArgs A;
  std::memset(&A, 0, sizeof(A));
  A.R = R;
  A.P = P;
  A.logp = logprobs;
  A.grad = grad_logits;
  A.partials = partials;
  MO_TRY(launch_slices(logits->dtype, A, sms, st));
  return launch_sums(partials, R.n, mid, sums, st);
}

size_t moteopt_preference_loss_workspace_size(const moteopt_logits* logits, int64_t sequences) {
  if (!shape_fits(logits) || sequences < 0) return 0;
  return preference_layout(logits->dtype, logits->seqs * logits->tokens, logits->vocab, sequences / 2).bytes;
}

int moteopt_preference_loss(const moteopt_logits* logits, const moteopt_positions* targets,
                            const moteopt_preference* preference, double temperature, float* loss, float* rewards,
                            float* logprobs, void* grad_logits, void* workspace, size_t workspace_bytes,
                            moteopt_stream_t stream) {
  const char* const who = "moteopt_preference_loss";
  Rows R;
  MO_TRY(check_logits(who, logits, targets, &R, temperature));
  if (!preference || !loss) return fail(MOTEOPT_ERR_INVALID, "moteopt_preference_loss: null pointer");
  const moteopt_preference& p = *preference;
  MO_TRY(check_divisor(who, p.divisor, p.divisor_device));
  if (p.sequences < 0 || p.sequences % 2 != 0 || p.sequences >= (int64_t{1} << 27))
    return fail(MOTEOPT_ERR_INVALID, "moteopt_preference_loss: the sequences are pairs: an even number of them");
  if (p.cu_seqlens ? logits->seqs != 1 : p.sequences != logits->seqs)
    return fail(MOTEOPT_ERR_INVALID, "moteopt_preference_loss: sequences do not match the logits");
  if (!std::isfinite(p.beta) || !(p.label_smoothing >= 0.0 && p.label_smoothing <= 1.0))
    return fail(MOTEOPT_ERR_INVALID, "moteopt_preference_loss: beta must be finite, label_smoothing in [0, 1]");
  if (p.sequences > 0 && (!rewards || !logprobs)) return fail(MOTEOPT_ERR_INVALID, "moteopt_preference_loss: null pointer");
  MO_TRY(check_aligned(who, 4, {loss, rewards, logprobs, p.cu_seqlens, p.ref_logprobs, p.divisor_device}));
  MO_TRY(check_aligned(who, esize(logits->dtype), {grad_logits}));
  const PreferenceLayout L = preference_layout(logits->dtype, R.n, R.vocab, p.sequences / 2);
  MO_TRY(check_ws(workspace, workspace_bytes, L.bytes));
  int sms = 0;
  MO_TRY(loss_setup(&sms));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (p.sequences == 0) {
    MO_CUDA(cudaMemsetAsync(loss, 0, sizeof(float), st));
    if (grad_logits && R.n > 0)
      MO_CUDA(cudaMemsetAsync(grad_logits, 0, static_cast<size_t>(R.n) * R.vocab * esize(logits->dtype), st));
    return MOTEOPT_OK;
  }
  char* const ws = static_cast<char*>(workspace);
  double* const logp64 = reinterpret_cast<double*>(ws + L.logp64);
  double* const lse = reinterpret_cast<double*>(ws + L.lse);
  float* const coef = reinterpret_cast<float*>(ws + L.coef);
  double* const pair_loss = reinterpret_cast<double*>(ws + L.pairs);
  R.cu = p.cu_seqlens;
  R.n_seqs = static_cast<int>(p.sequences);
  PairArgs A;
  std::memset(&A, 0, sizeof(A));
  A.R = R;
  A.pairs = static_cast<int>(p.sequences / 2);
  A.ref = p.ref_logprobs;
  A.beta = p.beta;
  A.eps = p.label_smoothing;
  A.inv_div = p.divisor_device ? 0.0 : 1.0 / p.divisor;
  A.div = p.divisor_device;
  A.average = p.average;
  A.logp64 = logp64;
  A.coef = grad_logits ? coef : nullptr;
  A.pair_loss = pair_loss;
  A.rewards = rewards;
  A.seq_logp = logprobs;
  Kept K;
  std::memset(&K, 0, sizeof(K));
  K.logp64 = logp64;
  K.lse64 = lse;
  K.coef_row = coef;
  K.pair_loss = pair_loss;
  K.pairs = A.pairs;
  K.loss = loss;
  const TileShape t = tile_shape(R.n, line_bytes(logits->dtype, R.vocab), sms);
  if (R.n > 0 && short_rows(logits->dtype, R.vocab) && one_cluster(R.n, t) && A.pairs <= kClusterPairs) {
    TileArgs B;
    std::memset(&B, 0, sizeof(B));
    B.R = R;
    B.logp64 = logp64;
    B.coef = coef;
    B.grad = grad_logits;
    B.K = K;
    B.pair = A;
    return launch_tile_cluster<kPreference>(logits->dtype, B, t, st);
  }
  if (R.n > 0)
    MO_TRY(launch_forward(logits->dtype, R, nullptr, nullptr, logp64, lse, coef, reinterpret_cast<Part*>(ws + L.parts), sms, st));
  MO_TRY(launch_after(pair_kernel, A, static_cast<unsigned>(A.pairs), kPairThreads, 0, st, "loss pair_kernel", R.n == 0));
  if (!grad_logits || R.n == 0) return launch_after(pair_sum_kernel, K, 1, 32, 0, st, "loss pair_sum_kernel");
  return launch_gradient(logits->dtype, R, K, grad_logits, sms, st, true);
}

}  // extern "C"
