// Softmax cross entropy of a dense head, without its logits: z = X W^T + b,
//     loss[m] = log sum_n exp z[m,n] - z[m,target[m]]        dz[m,n] = c[m] (exp(z[m,n] - lse[m]) - [n = target[m]])
//     dX = dz W      dW = dz^T X      db = sum over the rows of dz
//
// The forward is one product whose tiles leave, for each of their rows, the largest logit and the sum of the exponentials
// over it (DENSE_CE_STATS: 8 bytes for 512 of fp32 logits), which a second kernel joins to the row's log of the sum.
// The backward goes through the classes in pieces: a product makes a piece's logits again and leaves dz in the
// operands' type (DENSE_CE_GRAD, with the sums of db from unrounded values), two more take it to dX, which is added up in
// fp32 over the pieces, and to the piece's rows of dW.  8 M K N operations in all, 2 of them for what was not kept.
//
// The first piece's exponentials are kept where that takes less time than making them again: in the place of its
// dz, so in memory that the backward takes anyway, but held from the forward on, over the largest of 64: of bf16 operands in 16 bits
// (exp_code: within 2^-11 of each, and 2^-63, where rounding dz takes 2^-8), else as they are.  One pass then turns them into dz.
//
// Rows whose target is `ignore_index` count for nothing.  Of more than CE_ALL rows those that count are copied together first
// (a row is read and written once, against N products with it), and the products take their number from device
// memory: tiles and stages of rows that are not there end at once.  What ignored rows hold is never read then; of
// fewer rows it takes no part in a result either (their dz is 0 and their X is copied as zeros).
//
// A row's sum is kept apart from its target's exponential: with q = sum over the others of exp(z[m,n] - z[m,target]) the loss is
// log(1 + q) and dz at the target -c (1 - exp(-loss)), neither of which cancels in a row that is nearly certain.
//
// Bound by the products.  bf16, forward and backward: 8192 x 4096 over 131072 classes, a tenth of the rows ignored, 20.3 ms
// (statistics 7.2, dz 0.9 at 4.8 TB/s, dX 6.3, dW 5.8: up to 1.37 PFLOP/s of the rows that count); 4096 x 1024 over 50000 1.41
// (statistics 0.44 and 0.1 to keep exponentials, dz 0.16, dX 0.39, dW 0.36).  fp32 1024 x 1024 over 8192: 455 us.  The forward alone
// of 16 x 1024 over 32768: 17.4 us, where the weights take 13.5 at a copy's rate.
//
// Logits, sums and gradients are fp32 in units of log 2 behind the products (exp2 and log2 are the instructions); dz is rounded to
// the operands' type once, as the dense projection's.
#include "gl_dense.h"

namespace gl {

namespace {

// Rows above which ignored ones are left out of the products, which takes two launches more; of fewer rows all losses are one
// workgroup's work.  1024 features and 32768 classes, all rows and those that count: the forward alone of 64 rows 29 and
// 40 us, of 128 41 and 42, of 192 56 and 46; with the backward of 128 rows 120 and 135, of 192 150 and 144.
constexpr int CE_ALL = 128;
// Bytes of dz of a piece, unless the caller says otherwise: 1/72 of the card's memory.  16384 x 4096 over 131072 classes bf16, in
// pieces of 1, 2 and 4 GiB (that is whole): 47.1, 45.2 and 40.9 ms.
constexpr size_t CE_PIECE = 4ull << 30;
// Features from which exponentials are kept: the product that makes them again reads and multiplies that many, keeping them
// does not depend on it.  A training pass of 4096 rows, kept and not: bf16 and 50000 classes, 384 features 876 and 859 us,
// 512 935 and 952, 1024 1389 and 1581; fp32 and 16384 classes, 64 features 570 and 580, 512 1729 and 2133.
constexpr int CE_KEEP_BF16 = 512, CE_KEEP_F32 = 64;
constexpr float LN2 = 0.693147181f;

// what the forward keeps, in 32-bit words: rows that count, -, -, -; of every row that counts (in their order;
// of all rows where none is left out) the largest logit, the sum of the exponentials over it, and the loss; their rows; and of
// every row its place among them, or -1
struct Kept {
  int* count;
  float* top;
  float* sum;
  float* loss;
  int* index;
  int* rank;
};
Kept kept_of(int32_t* p, long long M) {
  float* f = (float*)p + 4;
  return Kept{p, f, f + M, f + 2 * M, p + 4 + 3 * M, p + 4 + 4 * M};
}

// ---- rows that count ---------------------------------------------------------------------------------------
// One workgroup, 4096 rows at a time; a thread has four neighbours.  8192 rows: 9 us.
__global__ __launch_bounds__(1024) void ce_index_kernel(const long long* __restrict__ target, long long M, long long ignored,
                                                        Kept k, float* __restrict__ loss) {
  __shared__ int waves[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0, turn = 0;
  for (long long m0 = 0; m0 < M; m0 += 4096, turn ^= 1) {
    const long long m = m0 + 4 * threadIdx.x;
    bool on[4];
    int before = 0, all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      on[j] = m + j < M && target[m + j] != ignored;
      const unsigned long long mask = __builtin_amdgcn_ballot_w64(on[j]);
      before += __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
      all += __builtin_popcountll(mask);
    }
    if (lane == 0) waves[turn][wave] = all;
    __syncthreads();  // (the other half is written when every thread has passed a barrier since it read this one)
    int at = base + before;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      const int c = waves[turn][w];
      at += w < wave ? c : 0;
      base += c;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (m + j >= M) break;
      k.rank[m + j] = on[j] ? at : -1;
      if (on[j]) k.index[at++] = (int)(m + j);
      else if (loss) loss[m + j] = 0.f;
    }
  }
  if (threadIdx.x == 0) *k.count = base;
}

// X's rows that count, to rows of padded(K) elements with zeros behind the last.  Of all rows (index null): those whose
// factor in `info` is 0 as zeros.  8 neighbours a thread, 4 rows a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void ce_gather_kernel(const T* __restrict__ X, long long sx, long long M, int K, const int* count,
                                                        const int* __restrict__ index, const uv4* __restrict__ info,
                                                        T* __restrict__ to) {
  const int ld = (K + 7) / 8 * 8, c0 = (blockIdx.y * 64 + (threadIdx.x & 63)) * 8;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= (index ? *count : M) || c0 >= ld) return;
  struct __attribute__((packed, aligned(2))) U { T x[8]; };
  T v[8];
  if (info && __uint_as_float(info[r][1]) == 0.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = T(0);
  } else {
    const T* src = X + (index ? index[r] : r) * sx;
    if (c0 + 8 <= K) {
      const U u = *reinterpret_cast<const U*>(src + c0);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = u.x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c0 + j < K ? src[c0 + j] : T(0);
    }
  }
  T* d = to + r * ld + c0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d[j] = v[j];
}
int launch_gather(const void* X, long long sx, long long M, int K, int es, const int* count, const int* index, const uv4* info,
                  void* to, hipStream_t s) {
  const dim3 grid((unsigned)((M + 3) / 4), (unsigned)ceil_div(padded(K), 512));
  if (es == 2) GL_LAUNCH(GL_KERNEL_CE_GATHER, ce_gather_kernel<unsigned short>, grid, dim3(256), 0, s, (const unsigned short*)X, sx, M, K, count, index, info, (unsigned short*)to);
  else GL_LAUNCH(GL_KERNEL_CE_GATHER, ce_gather_kernel<unsigned>, grid, dim3(256), 0, s, (const unsigned*)X, sx, M, K, count, index, info, (unsigned*)to);
  GL_CHECK_LAUNCH();
  return 0;
}

// ---- a row's loss --------------------------------------------------------------------------------------------
__device__ __forceinline__ float wave_max(float v) {
  auto up = [](float a, float b) { return __builtin_fmaxf(a, b); };
  v = up(v, dpp<0xB1>(v));
  v = up(v, dpp<0x4E>(v));
  v = up(v, dpp<0x141>(v));
  v = up(v, dpp<0x140>(v));
  return over_row<16>(v, up);
}
__device__ __forceinline__ float wave_add(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  v += dpp<0x140>(v);
  return over_row<16>(v, [](float a, float b) { return a + b; });
}
struct JoinK {
  const float* stats;
  const float* target_logit;
  const long long* target;
  long long M, ignored;
  int tiles, N, reduction;
  Kept k;
  float* loss;  // by row, or the result
};
// A row's statistics and loss, by a wave: every lane joins its tiles, then the lanes.  The loss is NaN where the target is no
// class, or a logit is +inf (infinity less infinity).
struct Row {
  float top, sum, loss;
};
__device__ __forceinline__ Row join_row(const JoinK& a, long long m, long long t) {
  const float* st = a.stats + 2 * m * a.tiles;
  float top = -__builtin_inff(), s = 0.f;
  for (int k = threadIdx.x & 63; k < a.tiles; k += 64) {
    const float x = st[2 * k], e = st[2 * k + 1], up = __builtin_fmaxf(top, x), ref = up == -__builtin_inff() ? 0.f : up;
    s = __builtin_fmaf(s, __builtin_amdgcn_exp2f(top - ref), e * __builtin_amdgcn_exp2f(x - ref));
    top = up;
  }
  const float up = wave_max(top), ref = up == -__builtin_inff() ? 0.f : up;
  s = wave_add(s * __builtin_amdgcn_exp2f(top - ref));
  const float nan = __builtin_nanf("");
  if (t < 0 || t >= a.N) return Row{up, s, nan};
  const float z = a.target_logit[m], q = s * __builtin_amdgcn_exp2f(up - z);
  if (z == __builtin_inff()) return Row{z, nan, nan};  // (the others' sum has seen every +inf but the target's)
  const Row r = z >= up ? Row{z, 1.f + q, 0.f} : Row{up, s + __builtin_amdgcn_exp2f(z - up), 0.f};
  return Row{r.top, r.sum, q > 1e6f ? (up - z + log2f(r.sum)) * LN2 : log1pf(q)};
}
// of rows that count, a wave each
__global__ __launch_bounds__(256) void ce_join_kernel(JoinK a) {
  const long long m = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= *a.k.count) return;
  const int row = a.k.index[m];
  const Row r = join_row(a, m, a.target[row]);
  if ((threadIdx.x & 63) != 0) return;
  a.k.top[m] = r.top;
  a.k.sum[m] = r.sum;
  a.k.loss[m] = r.loss;
  if (a.reduction == GL_CE_NONE) a.loss[row] = r.loss;
}
// The sum (in 64 bits) or the mean of the losses of rows that count; 0 of none.
__global__ __launch_bounds__(1024) void ce_sum_kernel(const float* __restrict__ rows, const int* count, int mean, float* loss) {
  __shared__ double sums[1024];
  const int n = *count;
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += (double)rows[i];
  sums[threadIdx.x] = s;
  for (int h = 512; h > 0; h >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < h) sums[threadIdx.x] += sums[threadIdx.x + h];
  }
  if (threadIdx.x == 0) *loss = (float)(mean && n > 0 ? sums[0] / n : sums[0]);
}
// Both, of up to CE_ALL rows of which none was left out, by one workgroup.
__global__ __launch_bounds__(1024) void ce_join_all_kernel(JoinK a) {
  __shared__ float losses[CE_ALL];
  __shared__ int counts[CE_ALL];
  for (long long m = threadIdx.x >> 6; m < a.M; m += 16) {
    const long long t = a.target[m];
    const bool on = t != a.ignored;
    const Row r = join_row(a, m, t);
    if ((threadIdx.x & 63) == 0) {
      const float loss = on ? r.loss : 0.f;
      a.k.top[m] = r.top;
      a.k.sum[m] = r.sum;
      a.k.loss[m] = loss;
      if (a.reduction == GL_CE_NONE) a.loss[m] = loss;
      losses[m] = loss;
      counts[m] = on;
    }
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  double s = 0.0;
  int n = 0;
  for (int m = 0; m < a.M; ++m) {
    s += (double)losses[m];
    n += counts[m];
  }
  *a.k.count = n;
  if (a.reduction != GL_CE_NONE) *a.loss = (float)(a.reduction == GL_CE_MEAN && n > 0 ? s / n : s);
}

// ---- backward ------------------------------------------------------------------------------------------------
// What a row's logits need to become dz, without the factor that all rows share (alpha: the mean's 1 / count and the
// upstream gradient, which the products' epilogues apply).  With it, the targets' dz, all near -alpha, would be rounded to bf16
// alike: up to 2^-9 of dX and dW as a whole.  (One that is no number stays with its rows: the others' gradients are 0.)  A target
// that is no class makes the row's dz NaN.
__global__ __launch_bounds__(256) void ce_info_kernel(const long long* __restrict__ target, long long M, long long ignored, int N,
                                                      int reduction, Kept k, bool all, const float* __restrict__ g, long long sg,
                                                      uv4* __restrict__ info, float* __restrict__ alpha) {
  const long long m = (long long)blockIdx.x * 256 + threadIdx.x;
  const int n = *k.count;
  const float shared = reduction == GL_CE_NONE ? 1.f : reduction == GL_CE_SUM ? *g : n > 0 ? *g / (float)n : 0.f;
  const bool number = __builtin_fabsf(shared) < __builtin_inff();
  if (m == 0) *alpha = number ? shared : 1.f;
  if (m >= (all ? M : n)) return;
  const long long row = all ? m : k.index[m], t = target[row];
  float c = reduction == GL_CE_NONE ? g[row * sg] : number ? 1.f : shared;
  if (t < 0 || t >= N) c = __builtin_nanf("");
  if (t == ignored) c = 0.f;
  info[m] = uv4{__float_as_uint(k.top[m]), __float_as_uint(c == 0.f ? 0.f : c / k.sum[m]), (unsigned)t, __float_as_uint(c * expm1f(-k.loss[m]))};
}

// dz of the columns whose exponentials were kept, in their place, and the sums of 64 rows of every column.  32 lanes of 8
// columns by 8 rows at a time, two rows of a lane in flight.
constexpr int CE_DZ_ROWS = 64;
template <bool BF>
__global__ __launch_bounds__(256) void ce_dz_kernel(void* exps, const float* __restrict__ tops, int N, long long M, const int* count,
                                                    const uv4* __restrict__ info, int first, float* __restrict__ part) {
  __shared__ float sums[8][256];
  const int ct = threadIdx.x & 31, rt = threadIdx.x >> 5, n = blockIdx.y * 256 + ct * 8;
  const long long pitch = (N + 7) & ~7, groups = (N + 63) >> 6;
  if (count && *count < M) M = *count;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (n < pitch) {
#pragma unroll 1
    for (int i = 0; i < CE_DZ_ROWS; i += 16) {
      float e[2][8], f[2];
      uv4 q[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const long long m = (long long)blockIdx.x * CE_DZ_ROWS + i + 8 * x + rt;
        if (m >= M) continue;
        q[x] = info[m];
        f[x] = tops[m * groups + (n >> 6)];
        if constexpr (BF) {
          const uv4 h = *reinterpret_cast<const uv4*>((const char*)exps + 2 * (m * pitch + n));
#pragma unroll
          for (int j = 0; j < 8; ++j) e[x][j] = exp_value(j & 1 ? h[j >> 1] >> 16 : h[j >> 1] & 0xffffu);
        } else {
          load8<false>(exps, m * pitch + n, 8, e[x]);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const long long m = (long long)blockIdx.x * CE_DZ_ROWS + i + 8 * x + rt;
        if (m >= M) continue;
        const float c = __uint_as_float(q[x][1]);
        const int t = (int)q[x][2] - first - n;
        f[x] = c * __builtin_amdgcn_exp2f(f[x] - __uint_as_float(q[x][0]));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[x][j] = c == 0.f || n + j >= N ? 0.f : t == j ? __uint_as_float(q[x][3]) : f[x] * e[x][j];
          s[j] += e[x][j];
        }
        store8<BF>(exps, m * pitch + n, 8, e[x]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[rt][ct * 8 + j] = s[j];
  __syncthreads();
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= N) return;
  float t = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) t += sums[r][threadIdx.x];
  part[(long long)blockIdx.x * N + col] = t;
}

// dX by row from the sums by rows that count (rank null: by row); rows that do not: zeros.  8 neighbours a thread.
template <bool FBF, bool TBF>
__global__ __launch_bounds__(256) void ce_scatter_kernel(const void* __restrict__ from, const int* __restrict__ rank, long long M,
                                                         int K, void* __restrict__ to) {
  const long long m = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int c = (blockIdx.y * 64 + (threadIdx.x & 63)) * 8;
  if (m >= M || c >= K) return;
  const long long r = rank ? rank[m] : m;
  float v[8];
  load8<FBF>(from, r * K + c, r < 0 ? 0 : K - c, v);
  store8<TBF>(to, m * K + c, K - c, v);
}

// ---- plans ---------------------------------------------------------------------------------------------------
bool dtype_ok(int d) { return d == GL_DTYPE_F32 || d == GL_DTYPE_BF16; }
bool on_element(const void* p, int dtype) { return ((uintptr_t)p & (uintptr_t)(es_of(dtype) - 1)) == 0; }
bool row_ok(long long stride, long long rows, long long cols) { return rows <= 1 || stride >= cols; }
constexpr long long CE_MOST_ROWS = 1LL << 24;  // rows' numbers and those of launches' workgroups are 32-bit

int check(const void* X, long long sx, const void* W, long long sw, const void* bias, const int64_t* target, long long M, int N, int K,
          int dtype, int reduction) {
  if (M < 0 || N < 1 || K < 1 || reduction < GL_CE_NONE || reduction > GL_CE_SUM) return GL_ERR_ARG;
  if (N > GL_DENSE_MAX_FEATURES || K > GL_DENSE_MAX_FEATURES || M > CE_MOST_ROWS || !dtype_ok(dtype)) return GL_ERR_UNSUPPORTED;
  if (M == 0) return 0;
  if (!X || !W || !target || ((uintptr_t)target & 7)) return GL_ERR_ARG;
  if (!row_ok(sx, M, K) || !row_ok(sw, N, K)) return GL_ERR_ARG;
  if (!on_element(X, dtype) || !on_element(W, dtype) || !on_element(bias, dtype)) return GL_ERR_ARG;
  return 0;
}
struct Layout {
  size_t at = 0;
  size_t take(size_t bytes) {
    const size_t p = at;
    at += (size_t)round_up((long long)bytes, 256);
    return p;
  }
};

// Classes of a piece: pieces of one size, in columns of the widest tiles, whose dz fits the budget (256 at least).
long long piece_of(long long M, int N, int dtype, size_t budget) {
  const long long fit = (long long)((budget ? budget : CE_PIECE) / ((size_t)M * es_of(dtype)));
  if (fit >= padded(N)) return N;
  const long long most = fit < 256 ? 256 : fit / 256 * 256, pieces = (N + most - 1) / most;
  const long long even = round_up((N + pieces - 1) / pieces, 256);
  return even < N ? even : N;
}
// Classes whose exponentials are kept: the first piece, unless the product that makes them again is short.
int kept_classes(long long M, int N, int K, int dtype, size_t budget) {
  return K >= (dtype == GL_DTYPE_BF16 ? CE_KEEP_BF16 : CE_KEEP_F32) ? (int)piece_of(M, N, dtype, budget) : 0;
}
size_t exps_at_tops(long long M, int cols, int dtype) { return (size_t)round_up(M * padded(cols) * es_of(dtype), 256); }
size_t exps_bytes(long long M, int cols, int dtype) {
  return cols ? exps_at_tops(M, cols, dtype) + (size_t)round_up(M * ((cols + 63) / 64) * 4, 256) : 0;
}

struct CeFwd {
  bool all;
  Operand x, w;
  Product pr;
  size_t x_at, w_at, stats, logit, kept, bytes;
};
CeFwd plan_ce(const GlCeArgs* a) {
  CeFwd p{};
  const int es = es_of(a->dtype);
  p.all = a->M <= CE_ALL;
  p.x = operand(a->X, a->sx, a->M, a->K, true, es);
  if (!p.all) p.x = Operand{nullptr, padded(a->K), a->M, a->K, true, true};
  p.w = operand(a->W, a->sw, a->N, a->K, true, es);
  p.pr = plan_product(a->dtype, a->M, a->N, a->K, 1);
  if (p.pr.splits == 0) return p;
  Layout l;
  p.x_at = l.take(copy_bytes(p.x, es));
  p.w_at = l.take(copy_bytes(p.w, es));
  p.stats = l.take((size_t)a->M * p.pr.tiles_n * 8);
  p.logit = l.take((size_t)a->M * 4);
  p.kept = l.take(a->kept ? 0 : GL_CE_KEPT_WORDS(a->M) * 4);
  p.bytes = l.at;
  return p;
}

DenseRowsK rows_product(int dtype, const Operand& x, const Operand& w, const Product& pl, const DenseEpi& e) {
  DenseRowsK k{};
  const int es = es_of(dtype);
  k.P = x.p;
  k.Q = w.p;
  k.ldp = x.ld * es;
  k.ldq = w.ld * es;
  k.R = x.cols;
  k.tiles_m = pl.tiles_m;
  k.tiles_n = pl.tiles_n;
  k.steps = pl.steps;
  k.steps_per_split = pl.steps_per_split;
  k.e = e;
  return k;
}
int launch_rows(int dtype, int kind, const Product& pl, const DenseRowsK& k, hipStream_t s) {
  return dtype == GL_DTYPE_BF16 ? launch_rows_tile_bf16(kind, DENSE_NT, pl.tile, k, 1, s)
                                : launch_rows_tile_f32(kind, DENSE_NT, pl.tile, k, 1, s);
}
// waves of a tile along its rows (gl_ce_bf16.hip, gl_ce_f32.hip): each leaves its own sums of db
int waves_m(int dtype, int tile) { return tile == (dtype == GL_DTYPE_BF16 ? DENSE_256X128 : DENSE_128_DEEP) ? 4 : 2; }

struct CeBwd {
  bool all;
  long long piece, pieces;  // classes of a piece
  Operand w;
  bool direct;              // dX's product writes dX itself
  int kept;                 // classes whose exponentials were kept: the first piece, or none
  size_t x_at, w_at, info, alpha, dz, dx, part, cols, bytes;
};
// the products of the classes [n0, n0 + n); dW's rows behind `head` go through one of their own
struct Piece {
  Product logits, px, pw, pw_tail;
  long long head;
};
Piece plan_piece(const GlCeBwdArgs* a, long long n) {
  Piece p{};
  p.head = n;
  p.logits = plan_product(a->dtype, a->M, (int)n, a->K, 1);
  if (a->dX) p.px = plan_product(a->dtype, a->M, a->K, n);
  if (a->dW) {
    p.pw = plan_product(a->dtype, n, a->K, a->M);
    // Tiles come in rounds of one a CU, and a last round of few takes as long as a full one.  The rows of whole rounds and
    // the rest as two products, where that is expected to take less: 50000 x 1024 over 4096, 784 tiles of 256 x 256 in 3.06
    // rounds, 429 us; as two 388.
    const long long per_row = (a->K + DENSE_BN[DENSE_256] - 1) / DENSE_BN[DENSE_256];
    const long long tiles = (n + 255) / 256 * per_row, head = tiles / 256 * 256 / per_row * 256;
    if (p.pw.splits && head > 0 && head < n) {
      const Product h = plan_product(a->dtype, head, a->K, a->M), t = plan_product(a->dtype, n - head, a->K, a->M);
      if (h.splits && t.splits && h.us + t.us < p.pw.us) {
        p.pw = h;
        p.pw_tail = t;
        p.head = head;
      }
    }
  }
  return p;
}
bool planned(const GlCeBwdArgs* a, const Piece& p) {
  return p.logits.splits && (!a->dX || p.px.splits) && (!a->dW || p.pw.splits);
}
int plan_ce_bwd(const GlCeBwdArgs* a, CeBwd* out) {
  CeBwd p{};
  const int es = es_of(a->dtype);
  p.all = a->M <= CE_ALL;
  p.piece = piece_of(a->M, a->N, a->dtype, a->piece_bytes);
  p.pieces = (a->N + p.piece - 1) / p.piece;
  p.w = operand(a->W, a->sw, a->N, a->K, true, es);
  p.direct = p.all && p.pieces == 1;
  size_t part = 0, cols = 0;
  for (int last = 0; last < 2; ++last) {
    const long long n = last ? a->N - (p.pieces - 1) * p.piece : p.piece;
    const Piece q = plan_piece(a, n);
    if (!planned(a, q)) return GL_ERR_UNSUPPORTED;
    const size_t c = (size_t)q.logits.tiles_m * waves_m(a->dtype, q.logits.tile) * n * 4;
    part = part > q.px.part_bytes ? part : q.px.part_bytes;
    part = part > q.pw.part_bytes ? part : q.pw.part_bytes;
    part = part > q.pw_tail.part_bytes ? part : q.pw_tail.part_bytes;
    cols = cols > c ? cols : c;
  }
  p.kept = a->exps ? kept_classes(a->M, a->N, a->K, a->dtype, a->piece_bytes) : 0;
  if (p.kept) {
    const size_t c = (size_t)((a->M + CE_DZ_ROWS - 1) / CE_DZ_ROWS) * p.kept * 4;
    cols = cols > c ? cols : c;
  }
  Layout l;
  p.x_at = l.take((size_t)a->M * padded(a->K) * es);
  p.w_at = l.take(copy_bytes(p.w, es));
  p.info = l.take((size_t)a->M * 16);
  p.alpha = l.take(4);
  p.dz = l.take(p.kept ? 0 : (size_t)a->M * padded(p.piece) * es);  // (later pieces' too take the first one's place)
  p.dx = l.take(a->dX && !p.direct ? (size_t)a->M * a->K * (p.pieces > 1 ? 4 : es) : 0);
  p.part = l.take(part);
  p.cols = l.take(a->db ? cols : 0);
  p.bytes = l.at;
  *out = p;
  return 0;
}

int check_bwd(const GlCeBwdArgs* a) {
  if (!a) return GL_ERR_ARG;
  GL_TRY(check(a->X, a->sx, a->W, a->sw, a->bias, a->target, a->M, a->N, a->K, a->dtype, a->reduction));
  if (!dtype_ok(a->g_dtype)) return GL_ERR_UNSUPPORTED;
  if (a->accumulate && a->g_dtype != GL_DTYPE_F32) return GL_ERR_ARG;
  if (a->M == 0) return 0;
  if (!a->kept || !a->dloss || ((uintptr_t)a->kept & 3) || ((uintptr_t)a->dloss & 3) || a->sdl < 0) return GL_ERR_ARG;
  if (!on_element(a->dX, a->dtype) || !on_element(a->dW, a->g_dtype) || !on_element(a->db, a->g_dtype) ||
      ((uintptr_t)a->exps & 255))
    return GL_ERR_ARG;
  return 0;
}
int check_fwd(const GlCeArgs* a) {
  if (!a) return GL_ERR_ARG;
  GL_TRY(check(a->X, a->sx, a->W, a->sw, a->bias, a->target, a->M, a->N, a->K, a->dtype, a->reduction));
  if (a->M == 0) return 0;
  if (!a->loss || ((uintptr_t)a->loss & 3) || ((uintptr_t)a->kept & 3) || ((uintptr_t)a->exps & 255) || (a->exps && !a->kept))
    return GL_ERR_ARG;
  return 0;
}

}  // namespace

}  // namespace gl

using namespace gl;

extern "C" int gl_ce_fwd_workspace(const GlCeArgs* a, size_t* bytes) {
  GL_TRY(check_fwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = 0;
  if (a->M == 0) return 0;
  const CeFwd p = plan_ce(a);
  if (p.pr.splits == 0) return GL_ERR_UNSUPPORTED;
  *bytes = p.bytes;
  return 0;
}

extern "C" int gl_ce_exps_bytes(const GlCeArgs* a, size_t* bytes) {
  GL_TRY(check_fwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = a->M == 0 ? 0 : exps_bytes(a->M, kept_classes(a->M, a->N, a->K, a->dtype, a->piece_bytes), a->dtype);
  return 0;
}

extern "C" int gl_ce_fwd(const GlCeArgs* a, void* stream) {
  GL_TRY(check_fwd(a));
  if (a->M == 0) return 0;
  CeFwd p = plan_ce(a);
  if (p.pr.splits == 0) return GL_ERR_UNSUPPORTED;
  if (a->ws_bytes < p.bytes) return GL_ERR_WORKSPACE;
  if (p.bytes && (!a->ws || ((uintptr_t)a->ws & 255))) return GL_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const int es = es_of(a->dtype);
  char* ws = (char*)a->ws;
  const Kept k = kept_of(a->kept ? a->kept : (int32_t*)(ws + p.kept), a->M);
  const long long* target = (const long long*)a->target;
  if (p.all) {
    GL_TRY(launch_align(&p.x, ws + p.x_at, &p.w, ws + p.w_at, es, s));
  } else {
    GL_LAUNCH(GL_KERNEL_CE_ROWS, ce_index_kernel, dim3(1), dim3(1024), 0, s, target, (long long)a->M, (long long)a->ignore_index, k,
              a->reduction == GL_CE_NONE ? a->loss : (float*)nullptr);
    GL_CHECK_LAUNCH();
    GL_TRY(launch_gather(a->X, a->sx, a->M, a->K, es, k.count, k.index, nullptr, ws + p.x_at, s));
    p.x.p = ws + p.x_at;
    GL_TRY(launch_align(nullptr, nullptr, &p.w, ws + p.w_at, es, s));
  }
  DenseEpi e = store_epi(nullptr, 0, a->dtype, a->M, a->N, a->dtype, 0);
  e.bias = a->bias;
  DenseRowsK d = rows_product(a->dtype, p.x, p.w, p.pr, e);
  d.rows = p.all ? nullptr : k.count;
  d.target = target;
  d.index = p.all ? nullptr : k.index;
  d.target_logit = (float*)(ws + p.logit);
  d.stats = (float*)(ws + p.stats);
  if (a->exps && (d.exps_cols = kept_classes(a->M, a->N, a->K, a->dtype, a->piece_bytes)) > 0) {
    d.exps = a->exps;
    d.exps_top = (float*)((char*)a->exps + exps_at_tops(a->M, d.exps_cols, a->dtype));
  }
  GL_TRY(launch_rows(a->dtype, DENSE_CE_STATS, p.pr, d, s));
  JoinK j{d.stats, d.target_logit, target, a->M, a->ignore_index, p.pr.tiles_n, a->N, a->reduction, k, a->loss};
  if (p.all) {
    GL_LAUNCH(GL_KERNEL_CE_ROWS, ce_join_all_kernel, dim3(1), dim3(1024), 0, s, j);
  } else {
    GL_LAUNCH(GL_KERNEL_CE_ROWS, ce_join_kernel, dim3((unsigned)((a->M + 3) / 4)), dim3(256), 0, s, j);
    GL_CHECK_LAUNCH();
    if (a->reduction != GL_CE_NONE)
      GL_LAUNCH(GL_KERNEL_CE_ROWS, ce_sum_kernel, dim3(1), dim3(1024), 0, s, (const float*)k.loss, (const int*)k.count,
                (int)(a->reduction == GL_CE_MEAN), a->loss);
  }
  GL_CHECK_LAUNCH();
  return 0;
}

extern "C" int gl_ce_bwd_workspace(const GlCeBwdArgs* a, size_t* bytes) {
  GL_TRY(check_bwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = 0;
  if (a->M == 0) return 0;
  CeBwd p;
  GL_TRY(plan_ce_bwd(a, &p));
  *bytes = p.bytes;
  return 0;
}

extern "C" int gl_ce_bwd(const GlCeBwdArgs* a, void* stream) {
  GL_TRY(check_bwd(a));
  if (a->M == 0 || (!a->dX && !a->dW && !a->db)) return 0;
  CeBwd p;
  GL_TRY(plan_ce_bwd(a, &p));
  if (a->ws_bytes < p.bytes) return GL_ERR_WORKSPACE;
  if (!a->ws || ((uintptr_t)a->ws & 255)) return GL_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const int es = es_of(a->dtype);
  char* ws = (char*)a->ws;
  const Kept k = kept_of(const_cast<int32_t*>(a->kept), a->M);
  uv4* info = (uv4*)(ws + p.info);
  GL_LAUNCH(GL_KERNEL_CE_ROWS, ce_info_kernel, dim3((unsigned)((a->M + 255) / 256)), dim3(256), 0, s, (const long long*)a->target,
            (long long)a->M, (long long)a->ignore_index, a->N, a->reduction, k, p.all, a->dloss, (long long)a->sdl, info, (float*)(ws + p.alpha));
  GL_CHECK_LAUNCH();
  const int* count = p.all ? nullptr : k.count;
  const float* alpha = a->reduction == GL_CE_NONE ? nullptr : (const float*)(ws + p.alpha);
  GL_TRY(launch_gather(a->X, a->sx, a->M, a->K, es, k.count, p.all ? nullptr : k.index, p.all ? info : nullptr, ws + p.x_at, s));
  GL_TRY(launch_align(nullptr, nullptr, &p.w, ws + p.w_at, es, s));
  const Operand x_rows{ws + p.x_at, padded(a->K), a->M, a->K, true, true};
  float* cols = (float*)(ws + p.cols);
  for (long long i = 0; i < p.pieces; ++i) {
    const long long n0 = i * p.piece, n = a->N - n0 < p.piece ? a->N - n0 : p.piece;
    const Piece q = plan_piece(a, n);
    const long long pitch = padded(n);
    Operand w = p.w;
    w.p = (const char*)w.p + n0 * w.ld * es;
    w.rows = n;
    void* at = p.kept ? a->exps : ws + p.dz;
    long long chunks;
    if (i == 0 && p.kept) {
      const dim3 grid((unsigned)((a->M + CE_DZ_ROWS - 1) / CE_DZ_ROWS), (unsigned)ceil_div(n, 256));
      const float* tops = (const float*)((char*)a->exps + exps_at_tops(a->M, p.kept, a->dtype));
      if (es == 2) GL_LAUNCH(GL_KERNEL_CE_GRAD, ce_dz_kernel<true>, grid, dim3(256), 0, s, at, tops, (int)n, (long long)a->M, count, (const uv4*)info, 0, a->db ? cols : (float*)nullptr);
      else GL_LAUNCH(GL_KERNEL_CE_GRAD, ce_dz_kernel<false>, grid, dim3(256), 0, s, at, tops, (int)n, (long long)a->M, count, (const uv4*)info, 0, a->db ? cols : (float*)nullptr);
      GL_CHECK_LAUNCH();
      chunks = grid.x;
    } else {
      DenseEpi e = store_epi(at, pitch, a->dtype, a->M, (int)n, a->dtype, 0);
      e.bias = a->bias ? (const char*)a->bias + n0 * es : nullptr;
      DenseRowsK d = rows_product(a->dtype, x_rows, w, q.logits, e);
      d.rows = count;
      d.row_info = info;
      d.first = (int)n0;
      d.col_sums = a->db ? cols : nullptr;
      d.pitch = (int)pitch;
      GL_TRY(launch_rows(a->dtype, DENSE_CE_GRAD, q.logits, d, s));
      chunks = (long long)q.logits.tiles_m * waves_m(a->dtype, q.logits.tile);
    }
    const Operand dz{at, pitch, a->M, (int)n, true, true};
    if (a->db) GL_TRY(launch_db(cols, chunks, (int)n, (char*)a->db + n0 * es_of(a->g_dtype), a->g_dtype, a->accumulate, s, alpha));
    if (a->dX) {
      const int to = p.pieces > 1 ? GL_DTYPE_F32 : a->dtype;
      GL_TRY(run_product(a->dtype, DENSE_NN, dz, w, n, q.px, ws + p.part,
                         store_epi(p.direct ? a->dX : ws + p.dx, a->K, to, a->M, a->K, a->dtype, i > 0), s, count, alpha));
    }
    for (long long from = 0, rows = q.head; a->dW && rows > 0; from += rows, rows = from < n ? n - from : 0) {
      Operand dz_t = dz;
      dz_t.p = (const char*)at + from * es;
      dz_t.cols = (int)rows;
      GL_TRY(run_product(a->dtype, DENSE_TN, dz_t, x_rows, a->M, from ? q.pw_tail : q.pw, ws + p.part,
                         store_epi((char*)a->dW + (n0 + from) * a->K * es_of(a->g_dtype), a->K, a->g_dtype, rows, a->K, a->dtype,
                                   a->accumulate), s, count, alpha));
    }
  }
  if (a->dX && !p.direct) {
    const dim3 grid((unsigned)((a->M + 3) / 4), (unsigned)ceil_div(a->K, 512));
    const int* rank = p.all ? nullptr : k.rank;
    const void* from = ws + p.dx;
    const bool bf = a->dtype == GL_DTYPE_BF16;
    if (!bf) GL_LAUNCH(GL_KERNEL_CE_ROWS, (ce_scatter_kernel<false, false>), grid, dim3(256), 0, s, from, rank, (long long)a->M, a->K, a->dX);
    else if (p.pieces > 1) GL_LAUNCH(GL_KERNEL_CE_ROWS, (ce_scatter_kernel<false, true>), grid, dim3(256), 0, s, from, rank, (long long)a->M, a->K, a->dX);
    else GL_LAUNCH(GL_KERNEL_CE_ROWS, (ce_scatter_kernel<true, true>), grid, dim3(256), 0, s, from, rank, (long long)a->M, a->K, a->dX);
    GL_CHECK_LAUNCH();
  }
  return 0;
}
