// The dense projection's entry points: plans, the kernels around the products, launches.
#include "gl_dense.h"

namespace gl {

namespace {

constexpr int es_of(int dtype) { return dtype == GL_DTYPE_BF16 ? 2 : 4; }
inline long long padded(long long n) { return round_up(n, 8); }  // row of a copied or computed operand

// ---- rows at 16-byte addresses --------------------------------------------------------------------
// The tile kernel loads 16 bytes at a time straight into LDS.  An operand whose rows do not start at
// 16-byte addresses, or (reduction along the row) end inside 16 bytes, is copied to rows of padded(cols)
// elements first, zeros behind the last: one pass over an operand that the product reads many times.
// Up to two operands a launch (blockIdx.z).
struct AlignK {
  const void* src[2];
  void* dst[2];
  long long ld[2], rows[2];
  int cols[2];
};
template <typename T>
__global__ __launch_bounds__(256) void dense_align_kernel(AlignK a) {
  const int z = blockIdx.z, cols = a.cols[z], ldd = (cols + 7) / 8 * 8;
  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), ld = a.ld[z];
  const int c0 = (blockIdx.y * 64 + (threadIdx.x & 63)) * 8;
  if (r >= a.rows[z] || c0 >= ldd) return;
  const T* src = (const T*)a.src[z];
  T v[8];
  if (c0 + 8 <= cols) {
    struct __attribute__((packed, aligned(2))) U { T x[8]; };
    const U u = *reinterpret_cast<const U*>(src + r * ld + c0);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = u.x[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c0 + j < cols ? src[r * ld + c0 + j] : T(0);
  }
  T* d = (T*)a.dst[z] + r * ldd + c0;
#pragma unroll
  for (int j = 0; j < 8; ++j) d[j] = v[j];
}

struct Operand {
  const void* p;
  long long ld;  // elements
  long long rows;
  int cols;
  bool rc;       // reduction along the row
  bool copied;   // through workspace
};
// Whether the tile kernel takes the operand as it is.  Its 32-bit offsets span 256 rows.
inline bool in_place(const Operand& o, int es) {
  const long long ldb = o.ld * es;
  return ((uintptr_t)o.p & 15) == 0 && (o.rows == 1 || ldb % 16 == 0) && (!o.rc || (long long)o.cols * es % 16 == 0) &&
         ldb * 256 < (1LL << 31);
}
inline Operand operand(const void* p, long long ld, long long rows, int cols, bool rc, int es) {
  Operand o{p, rows == 1 ? cols : ld, rows, cols, rc, false};
  if (!in_place(o, es)) o.copied = true;
  if (rows == 1) o.ld = padded(cols);  // never stepped along; keeps the buffer's size whole
  return o;
}
inline size_t copy_bytes(const Operand& o, int es) {
  return o.copied ? (size_t)round_up(o.rows * padded(o.cols) * es, 256) : 0;
}

// copies those of the operands (null or not) that need it to their places; they then are the copies
int launch_align(Operand* o0, void* dst0, Operand* o1, void* dst1, int es, hipStream_t s) {
  AlignK k{};
  int n = 0, cols = 0;
  long long rows = 0;
  Operand* const ops[2] = {o0, o1};
  void* const dst[2] = {dst0, dst1};
  for (int i = 0; i < 2; ++i) {
    Operand* o = ops[i];
    if (!o || !o->copied) continue;
    k.src[n] = o->p;
    k.dst[n] = dst[i];
    k.ld[n] = o->ld;
    k.rows[n] = o->rows;
    k.cols[n] = o->cols;
    rows = o->rows > rows ? o->rows : rows;
    cols = o->cols > cols ? o->cols : cols;
    ++n;
    o->p = dst[i];
    o->ld = padded(o->cols);
  }
  if (n == 0) return 0;
  const dim3 grid((unsigned)((rows + 3) / 4), (unsigned)ceil_div(padded(cols), 512), (unsigned)n);
  if (es == 2) GL_LAUNCH(GL_KERNEL_DENSE_ALIGN, dense_align_kernel<unsigned short>, grid, dim3(256), 0, s, k);
  else GL_LAUNCH(GL_KERNEL_DENSE_ALIGN, dense_align_kernel<unsigned>, grid, dim3(256), 0, s, k);
  GL_CHECK_LAUNCH();
  return 0;
}

// ---- the sums of a split product --------------------------------------------------------------------
// A lane holds 4 neighbouring columns and adds the splits in their order, then the epilogue.  Bound by the sums'
// bytes: 2 x 2048 x 1024 fp32 in 5.7 us (4.4 TB/s).
__global__ __launch_bounds__(256) void dense_join_kernel(const float* __restrict__ part, int splits, DenseEpi e) {
  const long long m = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int l = threadIdx.x & 63, n = blockIdx.y * 256 + l * 4, there = m < e.M ? e.N - n : 0;
  float v[1][4] = {{0.f, 0.f, 0.f, 0.f}}, b[4];
  dense_bias(e, n, b);
  const Added added = dense_added(e);
  uv4 r = {0u, 0u, 0u, 0u};
  if (added.p && there > 0) r = load_added(added.p + m * added.step + (long long)n * (added.bf ? 2 : 4), added.bf, there);
  if (there > 0) {
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      float t[4];
      load4(part, false, ((long long)s * e.M + m) * e.N + n, there, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[0][j] += t[j];
    }
  }
  dense_forward<1>(e, m, 1, n, v, b);
  if (added.p) add_added(v[0], r, added.bf);
  if (there > 0) store4(e.C, e.c_bf, m * e.sc + n, there, v[0]);
}

// ---- plan of a product --------------------------------------------------------------------------------
struct Product {
  double us;  // what the plan expects
  int tile, splits, steps_per_split, steps, tiles_m, tiles_n;
  size_t part_bytes;
};
// What a tile costs, measured on whole problems of 16 to 256 stages: workgroups of a CU, microseconds of a stage
// with one of them on each CU and with all, and of a tile's start and end.
struct TileCost {
  int per_cu;
  double alone, full, ends;
};
constexpr TileCost COST_BF16[DENSE_TILES] = {
    {1, 1.55, 1.55, 9}, {1, 0.88, 0.88, 7}, {2, 0.74, 1.05, 6}, {1, 0.57, 0.57, 6}, {2, 0.30, 0.68, 5}};
constexpr TileCost COST_F32[DENSE_TILES] = {
    {0, 0, 0, 0}, {0, 0, 0, 0}, {2, 2.15, 4.25, 6}, {1, 1.96, 1.96, 6}, {2, 1.10, 2.20, 5}};

// Tile and splits of the reduction: the least of rounds x (stages x cost + ends), no less than the operands' bytes
// take, plus for a split product its partial sums written and read (4 TB/s) and the launch that joins them.
Product plan_product(int dtype, long long M, int N, long long R) {
  constexpr int CUS = 256;
  constexpr long long MAX_BLOCKS = 1LL << 23;  // a launch has fewer than 2^32 threads
  const TileCost* cost = dtype == GL_DTYPE_BF16 ? COST_BF16 : COST_F32;
  Product best{};
  double best_t = 0;
  const long long steps = (R * es_of(dtype) + DENSE_BK - 1) / DENSE_BK;
  const double floor = (double)(M + N) * R * es_of(dtype) / 5.2e6;  // the operands' bytes
  for (int t = 0; t < DENSE_TILES; ++t) {
    const long long tm = (M + DENSE_BM[t] - 1) / DENSE_BM[t], tn = (N + DENSE_BN[t] - 1) / DENSE_BN[t];
    if (!cost[t].per_cu) continue;
    for (long long s = 1; s <= 32 && s <= steps; s = s < 4 ? s + 1 : s * 2) {
      const long long per = (steps + s - 1) / s, n = tm * tn * s, slots = CUS * cost[t].per_cu;
      if ((steps + per - 1) / per != s || n >= MAX_BLOCKS) continue;
      const double stage = n <= CUS ? cost[t].alone : cost[t].full;
      double time = (double)((n + slots - 1) / slots) * ((double)per * stage + cost[t].ends);
      if (time < floor) time = floor;
      if (s > 1) time += 4.0 + 0.15 * s + (double)s * M * N * 8 / 4.0e6;
      if (best_t == 0 || time < best_t) {
        best_t = time;
        best = Product{time, t, (int)s, (int)per, (int)steps, (int)tm, (int)tn, s > 1 ? (size_t)round_up(s * M * N * 4, 256) : 0};
      }
    }
  }
  return best;
}

int run_product(int dtype, int form, const Operand& p, const Operand& q, long long R, const Product& pl, void* part,
                const DenseEpi& e, hipStream_t s) {
  const int es = es_of(dtype);
  DenseK k{};
  k.P = p.p;
  k.Q = q.p;
  k.ldp = p.ld * es;
  k.ldq = q.ld * es;
  k.R = R;
  k.tiles_m = pl.tiles_m;
  k.tiles_n = pl.tiles_n;
  k.steps = pl.steps;
  k.steps_per_split = pl.steps_per_split;
  k.part = pl.splits > 1 ? (float*)part : nullptr;
  k.e = e;
  GL_TRY(dtype == GL_DTYPE_BF16 ? launch_dense_tile_bf16(form, pl.tile, k, pl.splits, s)
                                : launch_dense_tile_f32(form, pl.tile, k, pl.splits, s));
  if (pl.splits > 1) {
    const dim3 grid((unsigned)((e.M + 3) / 4), (unsigned)ceil_div(e.N, 256));
    GL_LAUNCH(GL_KERNEL_DENSE_JOIN, dense_join_kernel, grid, dim3(256), 0, s, (const float*)part, pl.splits, e);
    GL_CHECK_LAUNCH();
  }
  return 0;
}

// ---- dz = dY act'(z) and the sums of its columns -------------------------------------------------------
constexpr int DZ_COLS = 256;  // of a workgroup: 32 lanes of 8 columns by 8 rows at a time
// Rows a lane has in flight: more of them leave fewer waves.  16384 x 4096 bf16 with z in 8 bits, 340 MB: 2 rows 68 us
// (5.0 TB/s), 4 rows 78, 8 rows 120; z as it was, 4096 x 4096: 2 and 4 rows 22, 8 rows 30.
constexpr int DZ_AHEAD = 2;
// rows of a workgroup: half where the whole would leave CUs without a workgroup
inline int dz_rows(long long M, int N) { return (M + 63) / 64 * ceil_div(N, DZ_COLS) >= 512 ? 64 : 32; }

// One pass over dY and what was kept; memory bound.  dz is rounded to the operands' type, which the matrix
// instructions of dX and dW take (half a step of bf16 an element, beside W's and X's own); db sums it unrounded in fp32.
// dz may be null (only the sums), part too (only dz).  Rows of dz are padded(N) apart, zeros behind N.
template <bool YBF, bool OBF, int KEEP>
__global__ __launch_bounds__(256) void dense_dz_kernel(const void* __restrict__ dY, long long sdy, const void* __restrict__ z,
                                                       const uint8_t* __restrict__ ze, long long M, int N,
                                                       int rows, void* __restrict__ dz, float* __restrict__ part) {
  __shared__ float sums[8][DZ_COLS];
  const int ct = threadIdx.x & 31, rt = threadIdx.x >> 5;
  const int n = blockIdx.y * DZ_COLS + ct * 8;
  const long long ldz = (N + 7) / 8 * 8;
  const int nblk = (N + 31) / 32;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (n < N) {
#pragma unroll 1
    for (int i = 0; i < rows; i += 8 * DZ_AHEAD) {
      const long long m0 = (long long)blockIdx.x * rows + i + rt;
      if (m0 >= M) break;
      float g[DZ_AHEAD][8], t[DZ_AHEAD][8];
      unsigned bits[DZ_AHEAD];
      uv2 codes[DZ_AHEAD];
      int ex[DZ_AHEAD];
#pragma unroll
      for (int x = 0; x < DZ_AHEAD; ++x) {
        const long long m = m0 + 8 * x;
        const int there = m < M ? N - n : 0;
        load8<YBF>(dY, m * sdy + n, there, g[x]);
        if constexpr (KEEP == GL_KEEP_SIGN) bits[x] = m < M ? ((const unsigned*)z)[m * nblk + (n >> 5)] >> (n & 31) : 0u;
        if constexpr (KEEP == GL_KEEP_Z) load8<OBF>(z, m * ldz + n, there, t[x]);
        if constexpr (KEEP == GL_KEEP_Z8) {
          codes[x] = uv2{0u, 0u};
          ex[x] = 1;
          if (m < M) {
            codes[x] = *reinterpret_cast<const uv2*>((const uint8_t*)z + (m * nblk * 32 + n));
            ex[x] = ze[m * nblk + (n >> 5)];
          }
        }
      }
#pragma unroll
      for (int x = 0; x < DZ_AHEAD; ++x) {
        const long long m = m0 + 8 * x;
        if constexpr (KEEP == GL_KEEP_SIGN) {
#pragma unroll
          for (int j = 0; j < 8; ++j) g[x][j] = (bits[x] >> j) & 1u ? g[x][j] : 0.f;
        } else if constexpr (KEEP != GL_KEEP_NONE) {
          const float st = KEEP == GL_KEEP_Z8 ? p8_step(ex[x]) : 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            g[x][j] *= dgelu_f(KEEP == GL_KEEP_Z8 ? p8_value(codes[x][j >> 2], j & 3, st) : t[x][j]);
          // columns behind N hold dY's 0, but a code of 0 is NaN in a block without numbers
          if (KEEP == GL_KEEP_Z8 && n + 8 > N)
#pragma unroll
            for (int j = 0; j < 8; ++j) g[x][j] = n + j < N ? g[x][j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += g[x][j];
        if (dz && m < M) store8<OBF>(dz, m * ldz + n, 8, g[x]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[rt][ct * 8 + j] = s[j];
  __syncthreads();
  const int c = blockIdx.y * DZ_COLS + threadIdx.x;
  if (c >= N) return;
  float t = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) t += sums[r][threadIdx.x];
  part[(long long)blockIdx.x * N + c] = t;
}

// db from the sums of `chunks` row blocks: 32 columns a workgroup, 32 rows of lanes, then LDS.  256 x 4096 sums: 6 us,
// the latency of 8 dependent loads.
__global__ __launch_bounds__(1024) void dense_db_kernel(const float* __restrict__ part, long long chunks, int N,
                                                        void* __restrict__ db, int g_bf, int accumulate) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
  float s = 0.f;
  if (n < N)
    for (long long i = r; i < chunks; i += 32) s += part[i * N + n];
  sums[r][c] = s;
  __syncthreads();
  if (r != 0 || n >= N) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) t += sums[i][c];
  if (g_bf) ((unsigned short*)db)[n] = to_bf16(t);
  else ((float*)db)[n] = accumulate ? ((float*)db)[n] + t : t;
}

bool dtype_ok(int d) { return d == GL_DTYPE_F32 || d == GL_DTYPE_BF16; }
bool on_element(const void* p, int dtype) { return ((uintptr_t)p & (uintptr_t)(es_of(dtype) - 1)) == 0; }
bool row_ok(long long stride, long long rows, long long cols) { return rows <= 1 || stride >= cols; }

// ---- forward --------------------------------------------------------------------------------------------
int check_fwd(const GlDenseArgs* a) {
  if (!a || a->M < 0 || a->N < 1 || a->K < 1) return GL_ERR_ARG;
  if (a->N > GL_DENSE_MAX_FEATURES || a->K > GL_DENSE_MAX_FEATURES || a->M >= GL_DENSE_MAX_ROWS) return GL_ERR_UNSUPPORTED;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->y_dtype) || (a->res && !dtype_ok(a->res_dtype))) return GL_ERR_UNSUPPORTED;
  if (a->act < GL_ACT_IDENTITY || a->act > GL_ACT_GELU || a->keep < GL_KEEP_NONE || a->keep > GL_KEEP_Z8) return GL_ERR_ARG;
  if (a->M == 0) return 0;
  if (!a->X || !a->W || !a->Y || (a->keep != GL_KEEP_NONE && !a->z) || (a->keep == GL_KEEP_Z8 && !a->z_exp)) return GL_ERR_ARG;
  if (!row_ok(a->sx, a->M, a->K) || !row_ok(a->sw, a->N, a->K) || !row_ok(a->sy, a->M, a->N)) return GL_ERR_ARG;
  if (a->res && a->sr != 0 && !row_ok(a->sr, a->M, a->N)) return GL_ERR_ARG;
  if (!on_element(a->X, a->dtype) || !on_element(a->W, a->dtype) || !on_element(a->bias, a->dtype) ||
      !on_element(a->Y, a->y_dtype) || (a->res && !on_element(a->res, a->res_dtype)) || ((uintptr_t)a->z & 15))
    return GL_ERR_ARG;
  return 0;
}
struct FwdPlan {
  bool few;
  Operand x, w;
  Product pr;
  size_t off_w, off_part, bytes;
};
FwdPlan plan_fwd(const GlDenseArgs* a) {
  FwdPlan p{};
  const int es = es_of(a->dtype);
  p.x = operand(a->X, a->sx, a->M, a->K, true, es);
  p.w = operand(a->W, a->sw, a->N, a->K, true, es);
  p.pr = plan_product(a->dtype, a->M, a->N, a->K);
  if (p.pr.splits == 0) return p;  // refused by the entry points
  if (a->M <= DENSE_FEW_ROWS && a->keep == GL_KEEP_NONE) {
    // Few rows: a workgroup's 16 features' weights at 25 bytes a ns of a CU, and 5 TB/s in all, then X from L2 at
    // 40 bytes a ns; against the tiles and the copies they need.  4096 x 4096 bf16, in a graph: 1 row 6.9 us (tiles
    // 11.6), 16 rows 9.6 (12.3), 32 rows 13.8 (12.5), 64 rows 21.1 (12.7); from K 1024 64 rows 7.0 (8.4).
    const double row = (double)a->K * es, w = a->N * row, rounds = ceil_div(ceil_div(a->N, 16), 256);
    const double weights = w / 5.0e6 > rounds * 16 * row / 25e3 ? w / 5.0e6 : rounds * 16 * row / 25e3;
    const double few = 1.5 + weights + rounds * (double)a->M * row / 40e3;
    double tiles = p.pr.us;
    if (p.x.copied || p.w.copied) tiles += 3.0 + 2.0 * w / 4.0e6;
    if (few <= tiles) {
      p.few = true;
      return p;
    }
  }
  p.off_w = copy_bytes(p.x, es);
  p.off_part = p.off_w + copy_bytes(p.w, es);
  p.bytes = p.off_part + p.pr.part_bytes;
  return p;
}

// ---- backward ---------------------------------------------------------------------------------------------
int check_bwd(const GlDenseBwdArgs* a) {
  if (!a || a->M < 0 || a->N < 1 || a->K < 1) return GL_ERR_ARG;
  if (a->N > GL_DENSE_MAX_FEATURES || a->K > GL_DENSE_MAX_FEATURES || a->M >= GL_DENSE_MAX_ROWS) return GL_ERR_UNSUPPORTED;
  if (!dtype_ok(a->dtype) || !dtype_ok(a->dy_dtype) || !dtype_ok(a->g_dtype)) return GL_ERR_UNSUPPORTED;
  if (a->act < GL_ACT_IDENTITY || a->act > GL_ACT_GELU) return GL_ERR_ARG;
  const bool fits = a->act == GL_ACT_IDENTITY ? a->keep == GL_KEEP_NONE
                    : a->act == GL_ACT_RELU   ? a->keep == GL_KEEP_SIGN
                                              : (a->keep == GL_KEEP_Z || a->keep == GL_KEEP_Z8);
  if (!fits || (a->accumulate && a->g_dtype != GL_DTYPE_F32)) return GL_ERR_ARG;
  if (a->M == 0) return 0;
  if (!a->dY || (a->keep != GL_KEEP_NONE && !a->z) || (a->keep == GL_KEEP_Z8 && !a->z_exp)) return GL_ERR_ARG;
  if (a->dX && !a->W) return GL_ERR_ARG;
  if (a->dW && !a->X && (!a->xq || !a->xe)) return GL_ERR_ARG;
  if (!row_ok(a->sdy, a->M, a->N) || (a->X && !row_ok(a->sx, a->M, a->K)) || (a->W && !row_ok(a->sw, a->N, a->K)))
    return GL_ERR_ARG;
  if (!on_element(a->dY, a->dy_dtype) || !on_element(a->X, a->dtype) || !on_element(a->W, a->dtype) ||
      !on_element(a->dX, a->dtype) || !on_element(a->dW, a->g_dtype) || !on_element(a->db, a->g_dtype) ||
      ((uintptr_t)a->z & 15) || ((uintptr_t)a->xq & 7))
    return GL_ERR_ARG;
  return 0;
}
struct BwdPlan {
  bool own_dz;  // dz is written to workspace (else dY is dz as it stands)
  Operand dz_nn, dz_tn, w, x;
  Product px, pw;
  long long chunks;
  size_t off_x, off_w, off_part, off_db, bytes;
};
BwdPlan plan_bwd(const GlDenseBwdArgs* a) {
  BwdPlan p{};
  const int es = es_of(a->dtype);
  const long long ldz = padded(a->N);
  const bool products = a->dX || a->dW;
  p.dz_nn = Operand{a->dY, a->sdy, a->M, a->N, true, false};
  p.dz_tn = Operand{a->dY, a->sdy, a->M, a->N, false, false};
  if (a->M == 1) p.dz_nn.ld = p.dz_tn.ld = ldz;
  p.own_dz = products && (a->keep != GL_KEEP_NONE || a->dy_dtype != a->dtype || !in_place(p.dz_nn, es));
  size_t at = 0;
  if (p.own_dz) {
    p.dz_nn.ld = p.dz_tn.ld = ldz;
    at += (size_t)round_up(a->M * ldz * es, 256);
  }
  p.off_x = at;
  size_t part = 0;
  if (a->dW) {
    if (a->X) {
      p.x = operand(a->X, a->sx, a->M, a->K, false, es);
      at += copy_bytes(p.x, es);
    } else {
      p.x = Operand{nullptr, padded(a->K), a->M, a->K, false, false};
      at += (size_t)round_up(a->M * padded(a->K) * es, 256);
    }
    p.pw = plan_product(a->dtype, a->N, a->K, a->M);
    part = p.pw.part_bytes;
  }
  p.off_w = at;
  if (a->dX) {
    p.w = operand(a->W, a->sw, a->N, a->K, false, es);
    at += copy_bytes(p.w, es);
    p.px = plan_product(a->dtype, a->M, a->K, a->N);
    part = part > p.px.part_bytes ? part : p.px.part_bytes;
  }
  p.off_part = at;
  at += part;
  p.off_db = at;
  p.chunks = (a->M + dz_rows(a->M, a->N) - 1) / dz_rows(a->M, a->N);
  if (a->db) at += (size_t)round_up(p.chunks * a->N * 4, 256);
  p.bytes = at;
  return p;
}

template <bool YBF, bool OBF, int KEEP>
int launch_dz_as(const GlDenseBwdArgs* a, void* dz, float* part, hipStream_t s) {
  const int rows = dz_rows(a->M, a->N);
  const dim3 grid((unsigned)((a->M + rows - 1) / rows), (unsigned)ceil_div(a->N, DZ_COLS));
  GL_LAUNCH(GL_KERNEL_DENSE_DZ, (dense_dz_kernel<YBF, OBF, KEEP>), grid, dim3(256), 0, s, a->dY, a->sdy, a->z, a->z_exp,
            (long long)a->M, a->N, rows, dz, part);
  GL_CHECK_LAUNCH();
  return 0;
}
template <bool YBF, bool OBF>
int launch_dz_of(const GlDenseBwdArgs* a, void* dz, float* part, hipStream_t s) {
  if (a->keep == GL_KEEP_NONE) return launch_dz_as<YBF, OBF, GL_KEEP_NONE>(a, dz, part, s);
  if (a->keep == GL_KEEP_SIGN) return launch_dz_as<YBF, OBF, GL_KEEP_SIGN>(a, dz, part, s);
  if (a->keep == GL_KEEP_Z) return launch_dz_as<YBF, OBF, GL_KEEP_Z>(a, dz, part, s);
  return launch_dz_as<YBF, OBF, GL_KEEP_Z8>(a, dz, part, s);
}
int launch_dz(const GlDenseBwdArgs* a, void* dz, float* part, hipStream_t s) {
  const bool o = a->dtype == GL_DTYPE_BF16;
  if (a->dy_dtype == GL_DTYPE_BF16) return o ? launch_dz_of<true, true>(a, dz, part, s) : launch_dz_of<true, false>(a, dz, part, s);
  return o ? launch_dz_of<false, true>(a, dz, part, s) : launch_dz_of<false, false>(a, dz, part, s);
}

DenseEpi store_epi(void* C, long long sc, int c_dtype, long long M, int N, int op_dtype, int accumulate) {
  DenseEpi e{};
  e.C = C;
  e.sc = sc;
  e.M = M;
  e.N = N;
  e.act = GL_ACT_IDENTITY;
  e.keep = GL_KEEP_NONE;
  e.op_bf = op_dtype == GL_DTYPE_BF16;
  e.c_bf = c_dtype == GL_DTYPE_BF16;
  e.accumulate = accumulate;
  return e;
}

}  // namespace

}  // namespace gl

using namespace gl;

extern "C" int gl_dense_fwd_workspace(const GlDenseArgs* a, size_t* bytes) {
  GL_TRY(check_fwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = 0;
  if (a->M == 0) return 0;
  const FwdPlan p = plan_fwd(a);
  if (p.pr.splits == 0) return GL_ERR_UNSUPPORTED;
  *bytes = p.bytes;
  return 0;
}

extern "C" int gl_dense_fwd(const GlDenseArgs* a, void* stream) {
  GL_TRY(check_fwd(a));
  if (a->M == 0) return 0;
  FwdPlan p = plan_fwd(a);
  if (p.pr.splits == 0) return GL_ERR_UNSUPPORTED;
  if (a->ws_bytes < p.bytes) return GL_ERR_WORKSPACE;
  if (p.bytes && (!a->ws || ((uintptr_t)a->ws & 255))) return GL_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  DenseEpi e = store_epi(a->Y, a->sy, a->y_dtype, a->M, a->N, a->dtype, 0);
  e.bias = a->bias;
  e.res = a->res;
  e.sr = a->sr;
  e.res_bf = a->res_dtype == GL_DTYPE_BF16;
  e.z = a->z;
  e.ze = a->z_exp;
  e.act = a->act;
  e.keep = a->keep;
  if (p.few) return launch_dense_few(a, e, s);
  const int es = es_of(a->dtype);
  char* ws = (char*)a->ws;
  GL_TRY(launch_align(&p.x, ws, &p.w, ws + p.off_w, es, s));
  return run_product(a->dtype, DENSE_NT, p.x, p.w, a->K, p.pr, ws + p.off_part, e, s);
}

extern "C" int gl_dense_bwd_workspace(const GlDenseBwdArgs* a, size_t* bytes) {
  GL_TRY(check_bwd(a));
  if (!bytes) return GL_ERR_ARG;
  *bytes = 0;
  if (a->M == 0) return 0;
  const BwdPlan p = plan_bwd(a);
  if ((a->dX && p.px.splits == 0) || (a->dW && p.pw.splits == 0)) return GL_ERR_UNSUPPORTED;
  *bytes = p.bytes;
  return 0;
}

extern "C" int gl_dense_bwd(const GlDenseBwdArgs* a, void* stream) {
  GL_TRY(check_bwd(a));
  if (a->M == 0) return 0;
  BwdPlan p = plan_bwd(a);
  if ((a->dX && p.px.splits == 0) || (a->dW && p.pw.splits == 0)) return GL_ERR_UNSUPPORTED;
  if (a->ws_bytes < p.bytes) return GL_ERR_WORKSPACE;
  if (p.bytes && (!a->ws || ((uintptr_t)a->ws & 255))) return GL_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const int es = es_of(a->dtype);
  char* ws = (char*)a->ws;
  void* dz = p.own_dz ? ws : nullptr;
  float* db_part = a->db ? (float*)(ws + p.off_db) : nullptr;
  if (dz || db_part) GL_TRY(launch_dz(a, dz, db_part, s));
  if (a->db) {
    GL_LAUNCH(GL_KERNEL_DENSE_DB, dense_db_kernel, dim3((unsigned)ceil_div(a->N, 32)), dim3(1024), 0, s, (const float*)db_part,
              p.chunks, a->N, a->db, (int)(a->g_dtype == GL_DTYPE_BF16), a->accumulate);
    GL_CHECK_LAUNCH();
  }
  if (dz) p.dz_nn.p = p.dz_tn.p = dz;
  GL_TRY(launch_align(a->dW && a->X ? &p.x : nullptr, ws + p.off_x, a->dX ? &p.w : nullptr, ws + p.off_w, es, s));
  if (a->dX) {
    GL_TRY(run_product(a->dtype, DENSE_NN, p.dz_nn, p.w, a->N, p.px, ws + p.off_part,
                       store_epi(a->dX, a->K, a->dtype, a->M, a->K, a->dtype, 0), s));
  }
  if (a->dW) {
    if (!a->X) {
      GL_TRY(launch_unpack8(a->xq, a->xe, a->M, a->K, ws + p.off_x, p.x.ld, a->dtype, s));
      p.x.p = ws + p.off_x;
    }
    GL_TRY(run_product(a->dtype, DENSE_TN, p.dz_tn, p.x, a->M, p.pw, ws + p.off_part,
                       store_epi(a->dW, a->K, a->g_dtype, a->N, a->K, a->dtype, a->accumulate), s));
  }
  return 0;
}
