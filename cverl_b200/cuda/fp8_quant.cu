// Block-scaled 8-bit quantisation: one pass over a bf16 or fp32 matrix that writes its codes and scales in the row
// form, the transposed form, or both, and the same with one scale per 128 x 128 block for weights.
//
// Bound by HBM: 2 bytes read and 1 written per element and form (bf16), no arithmetic to speak of.  One CTA takes a
// 128 x 128 tile, the smallest piece that holds whole blocks of both forms: a thread keeps 8 rows x 8 columns in
// registers, a half-warp covers the 128 columns of a row (256 bytes a load), so a row block's maximum is four
// shuffles and a column block's is eight values per thread and one shared-memory maximum.  Both forms come from the
// registers of the one read; only the transposed codes pass through shared memory.
#include "fp8_common.cuh"
#include "fp8_launch.h"

namespace cvb {

// A kernel may be placed while the one before it in the stream still runs, and lets the next one be placed as soon as it
// may itself begin.  Ordinarily it begins when that has ended: all that was launched before is then complete, and its own
// loads are not of the read-only kind, which would allow them to be served from before that.  `beside`: it reads nothing
// that the launch before it writes, nor writes what that touches, and begins at once; it ends after it, so that what
// follows may rely on both.  1301 x 1000 with a weight of 520 rows, forward: 9.9 us, 12.3 one after the other.
template <typename Args>
static void launch_rows(void (*kernel)(const Args), const Args& p, long long grid, int threads, cudaStream_t s) {
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kernel, p);
}

constexpr int QT = 128;            // tile edge
constexpr int Q_THREADS = 256;

struct QuantArgs {
  const void* x;
  long long rows, cols, x_stride;
  int vec;                         // base and row stride are 16-byte aligned
  uint8_t *q, *sf;                 // row form
  long long q_ld;
  int kgroups;                     // ceil(ceil(cols / 128) / 4)
  uint8_t *qt, *sft;               // transposed form
  uint8_t *ps, *pst;               // scale bytes of each form in plain order [row, block]; may be null
  long long qt_ld;
  int kgroups_t;
  int col_tiles, beside;
  // values are x * rstd[row] * (w_offset + w[col]) where rstd is given
  const float* rstd;
  const __nv_bfloat16* w;
  float w_offset;
};

// A thread's 8 x 8 piece of the tile as it was read.  bf16 stays packed (32 registers), so that two CTAs with 64 KB
// of loads in flight fit an SM; values are formed where they are used, once for each form.
template <typename T, bool NORM>
struct Piece;

template <int FMT, typename P>
__device__ __forceinline__ uint2 fp8_row_codes(const P& x, int i, uint32_t inv) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = x.get(i, j);
  return fp8_pack8<FMT>(v, i & 1 ? fp8_high(inv) : fp8_low(inv));
}
template <int FMT, typename P>
__device__ __forceinline__ void fp8_column_codes(const P& x, int j, uint32_t inv, uint2 (&codes)[2]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x.get(i, j + c);
    codes[c] = fp8_pack8<FMT>(v, c ? fp8_high(inv) : fp8_low(inv));
  }
}

template <bool NORM>
struct Piece<__nv_bfloat16, NORM> {
  uint32_t raw[8][4];
  float rstd[NORM ? 8 : 1], gain[NORM ? 8 : 1];
  __device__ __forceinline__ void load(const QuantArgs& p, long long r0, long long c0, int nc) {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + r0 * p.x_stride + c0;
    if (p.vec && nc == 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (r0 + i < p.rows) u = *reinterpret_cast<const uint4*>(x + i * p.x_stride);
        raw[i][0] = u.x, raw[i][1] = u.y, raw[i][2] = u.z, raw[i][3] = u.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t* row = reinterpret_cast<const uint16_t*>(x + i * p.x_stride);
        const int n = r0 + i < p.rows ? nc : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          raw[i][j] = (2 * j < n ? row[2 * j] : 0u) | ((2 * j + 1 < n ? row[2 * j + 1] : 0u) << 16);
      }
    }
    if constexpr (NORM) {
      fp8_load8(p.w + c0, nc, (reinterpret_cast<uintptr_t>(p.w) & 15) == 0, gain);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        gain[i] += p.w_offset;       // columns and rows outside hold zeros: whatever they are multiplied by is finite
        rstd[i] = r0 + i < p.rows ? p.rstd[r0 + i] : 0.f;
      }
    }
  }
  // the packed words are what stays live from here on, not the values formed from them
  __device__ __forceinline__ void keep_packed() {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+r"(raw[i][0]), "+r"(raw[i][1]), "+r"(raw[i][2]), "+r"(raw[i][3]));
  }
  // get() with an index that is not known when compiling
  __device__ __forceinline__ float at(int i, int j) const {
    float v = 0.f;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (a == i && b == j) v = get(a, b);
    return v;
  }
  __device__ __forceinline__ float scaled(int i, int j) const {       // x, or x rstd
    const uint32_t w = raw[i][j >> 1];
    const float v = __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
    if constexpr (NORM) return v * rstd[i];
    else return v;
  }
  __device__ __forceinline__ float get(int i, int j) const {
    if constexpr (NORM) return scaled(i, j) * gain[j];
    else return scaled(i, j);
  }
  // codes of row i with the scale in the half i & 1 of `inv`; of columns j and j + 1 with those in its low and high half.
  // bf16 are scaled as they are read, two to an instruction: 20480 x 3584, both forms, 57.4 us, 59.7 value by value.
  template <int FMT>
  __device__ __forceinline__ uint2 row_codes(int i, uint32_t inv) const {
    if constexpr (NORM) return fp8_row_codes<FMT>(*this, i, inv);
    const uint32_t both = __byte_perm(inv, inv, i & 1 ? 0x3232 : 0x1010);
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = fp8_mul_bf16x2(raw[i][j], both);
      v[2 * j] = fp8_low(w), v[2 * j + 1] = fp8_high(w);
    }
    return make_uint2(fp8_pack4<FMT>(v[0], v[1], v[2], v[3]), fp8_pack4<FMT>(v[4], v[5], v[6], v[7]));
  }
  template <int FMT>
  __device__ __forceinline__ void column_codes(int j, uint32_t inv, uint2 (&codes)[2]) const {
    if constexpr (NORM) {
      fp8_column_codes<FMT>(*this, j, inv, codes);
    } else {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = fp8_mul_bf16x2(raw[i][j >> 1], inv);
        a[i] = fp8_low(w), b[i] = fp8_high(w);
      }
      codes[0] = make_uint2(fp8_pack4<FMT>(a[0], a[1], a[2], a[3]), fp8_pack4<FMT>(a[4], a[5], a[6], a[7]));
      codes[1] = make_uint2(fp8_pack4<FMT>(b[0], b[1], b[2], b[3]), fp8_pack4<FMT>(b[4], b[5], b[6], b[7]));
    }
  }
};

template <>
struct Piece<float, false> {
  float raw[8][8];
  __device__ __forceinline__ void load(const QuantArgs& p, long long r0, long long c0, int nc) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      fp8_load8(static_cast<const float*>(p.x) + (r0 + i) * p.x_stride + c0, r0 + i < p.rows ? nc : 0, p.vec, raw[i]);
  }
  __device__ __forceinline__ void keep_packed() {}
  __device__ __forceinline__ float at(int i, int j) const {
    float v = 0.f;
#pragma unroll
    for (int a = 0; a < 8; ++a)
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (a == i && b == j) v = raw[a][b];
    return v;
  }
  __device__ __forceinline__ float get(int i, int j) const { return raw[i][j]; }
  template <int FMT>
  __device__ __forceinline__ uint2 row_codes(int i, uint32_t inv) const { return fp8_row_codes<FMT>(*this, i, inv); }
  template <int FMT>
  __device__ __forceinline__ void column_codes(int j, uint32_t inv, uint2 (&codes)[2]) const {
    fp8_column_codes<FMT>(*this, j, inv, codes);
  }
};

// Maxima of the piece's rows and columns over finite values, two 16-bit maxima a word: rows 2i, 2i + 1 in rmax[i],
// columns 2j, 2j + 1 in cmax[j].  Returns whether a value was not finite.
template <typename T, bool NORM>
__device__ __forceinline__ bool piece_maxima(const Piece<T, NORM>& x, uint32_t (&rmax)[4], uint32_t (&cmax)[4]) {
  float rm[8], cm[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rm[i] = cm[i] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(x.get(i, j));
      rm[i] = fmaxf(rm[i], a);
      cm[j] = fmaxf(cm[j], a);
    }
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) all = fmaxf(all, rm[i]);
  const bool odd = __float_as_uint(all) >= 0x7F800000u;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rm[i] = cm[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = fabsf(x.get(i, j));
        if (__float_as_uint(a) < 0x7F800000u) {
          rm[i] = fmaxf(rm[i], a);
          cm[j] = fmaxf(cm[j], a);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    rmax[i] = fp8_max16(__float_as_uint(rm[2 * i])) | (fp8_max16(__float_as_uint(rm[2 * i + 1])) << 16);
    cmax[i] = fp8_max16(__float_as_uint(cm[2 * i])) | (fp8_max16(__float_as_uint(cm[2 * i + 1])) << 16);
  }
  return odd;
}

// The norm's result, columns alone (rmax is not written).  Rounding keeps the order of magnitudes, so a column's maximum
// of |x rstd gain| is the gain's product with that of |x rstd|; NaN, a gain's among them, is passed over by fmaxf.
__device__ __forceinline__ bool piece_maxima(const Piece<__nv_bfloat16, true>& x, uint32_t (&)[4], uint32_t (&cmax)[4]) {
  float cm[8], all = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    cm[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) cm[j] = fmaxf(cm[j], fabsf(x.scaled(i, j)));
    cm[j] = fmaxf(0.f, cm[j] * fabsf(x.gain[j]));
    all = fmaxf(all, cm[j]);
  }
  const bool odd = __float_as_uint(all) >= 0x7F800000u;
  if (odd) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cm[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x.get(i, j));
        if (__float_as_uint(a) < 0x7F800000u) cm[j] = fmaxf(cm[j], a);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    cmax[j] = fp8_max16(__float_as_uint(cm[2 * j])) | (fp8_max16(__float_as_uint(cm[2 * j + 1])) << 16);
  return odd;
}

// bf16 as read: magnitudes are compared as pairs of 16-bit integers, half the instructions of the above
__device__ __forceinline__ bool piece_maxima(const Piece<__nv_bfloat16, false>& x, uint32_t (&rmax)[4], uint32_t (&cmax)[4]) {
  uint32_t row[8], all = 0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) cmax[j] = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    row[i] = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t m = x.raw[i][j] & 0x7FFF7FFFu;
      row[i] = __vmaxu2(row[i], m);
      cmax[j] = __vmaxu2(cmax[j], m);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) all = __vmaxu2(all, cmax[j]);
  const bool odd = (all & 0xFFFFu) >= 0x7F80u || (all >> 16) >= 0x7F80u;
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) cmax[j] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t m = x.raw[i][j] & 0x7FFF7FFFu;
        if ((m & 0xFFFFu) >= 0x7F80u) m &= 0xFFFF0000u;
        if ((m >> 16) >= 0x7F80u) m &= 0xFFFFu;
        row[i] = __vmaxu2(row[i], m);
        cmax[j] = __vmaxu2(cmax[j], m);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)     // the larger half of each row's word: rows 2i and 2i + 1 side by side
    rmax[i] = __vmaxu2(__byte_perm(row[2 * i], row[2 * i + 1], 0x5410), __byte_perm(row[2 * i], row[2 * i + 1], 0x7632));
  return odd;
}

// Instructions bound this kernel before HBM does (71 % of the issue slots and 65 % of the integer pipe at 4.1 TB/s in
// an earlier form), so scales are computed two to a word, a column's once for the tile, addresses advance by a stride,
// and an infinity costs nothing where there is none.
template <typename T, int FMT, bool NORM, bool ROWS, bool COLS, bool BLOCK, int CTAS = sizeof(T) == 4 ? 1 : NORM ? 2 : 3>
__global__ void __launch_bounds__(Q_THREADS, CTAS)
fp8_quant_kernel(const QuantArgs p) {
  if (!p.beside) wait_for_previous_kernel();      // see launch_rows
  launch_dependents();
  __shared__ __align__(16) uint32_t s_max[COLS || BLOCK ? Q_THREADS / 32 : 1][QT / 2];   // column maxima by warp
  __shared__ __align__(16) uint32_t s_inv[COLS ? QT / 2 : 4];      // 2^-e of two columns a word, as bf16
  __shared__ __align__(16) uint8_t s_t[COLS ? QT * QT : 16];       // transposed codes, 8-byte units XOR-swizzled
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int cl = lane & 15, rg = warp * 2 + (lane >> 4);           // columns 8 cl .. + 7, rows 8 rg .. + 7 of the tile
  const int tile_r = blockIdx.x / p.col_tiles;
  const int tile_c = blockIdx.x - tile_r * p.col_tiles;
  const long long r0 = static_cast<long long>(tile_r) * QT + rg * 8;
  const long long c0 = static_cast<long long>(tile_c) * QT + cl * 8;
  const int nr = static_cast<int>(max(0ll, min(8ll, p.rows - r0))), nc = static_cast<int>(max(0ll, min(8ll, p.cols - c0)));
  Piece<T, NORM> x;
  x.load(p, r0, c0, nc);
  uint32_t rmax[4], cmax[4];
  const bool odd = piece_maxima(x, rmax, cmax);
  x.keep_packed();
  uint32_t tile_bytes = 0;      // BLOCK: the tile's scale in both halves
  if (BLOCK) {
    uint32_t m = __vmaxu2(__vmaxu2(rmax[0], rmax[1]), __vmaxu2(rmax[2], rmax[3]));
    m = __reduce_max_sync(0xffffffffu, max(m & 0xFFFFu, m >> 16));
    if (lane == 0) s_max[warp][0] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Q_THREADS / 32; ++w) m = max(m, s_max[w][0]);
    tile_bytes = fp8_scale_bytes<FMT>(m * 0x00010001u);
  } else if (COLS) {
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = __vmaxu2(cmax[j], __shfl_xor_sync(0xffffffffu, cmax[j], 16));
    if (lane < 16) *reinterpret_cast<uint4*>(&s_max[warp][cl * 4]) = make_uint4(c[0], c[1], c[2], c[3]);
    __syncthreads();
    if (threadIdx.x < QT / 2) {            // two columns a thread
      uint32_t m = s_max[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < Q_THREADS / 32; ++w) m = __vmaxu2(m, s_max[w][threadIdx.x]);
      const uint32_t bytes = fp8_scale_bytes<FMT>(m);
      s_inv[threadIdx.x] = fp8_inverse_scales(bytes);
      const long long col = static_cast<long long>(tile_c) * QT + threadIdx.x * 2;
      uint8_t* sf = p.sft + fp8_sf_offset(col, tile_r, p.kgroups_t);
      sf[0] = static_cast<uint8_t>(bytes);
      sf[16] = static_cast<uint8_t>(bytes >> 16);
      if (p.pst != nullptr) {
        const long long nb = (p.rows + QT - 1) / QT;
        if (col < p.cols) p.pst[col * nb + tile_r] = static_cast<uint8_t>(bytes);
        if (col + 1 < p.cols) p.pst[(col + 1) * nb + tile_r] = static_cast<uint8_t>(bytes >> 16);
      }
    }
  }
  if (ROWS) {
    if (!BLOCK) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) rmax[i] = __vmaxu2(rmax[i], __shfl_xor_sync(0xffffffffu, rmax[i], o));
    }
    uint32_t bytes[4], inv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bytes[i] = BLOCK ? tile_bytes : fp8_scale_bytes<FMT>(rmax[i]);
      inv[i] = fp8_inverse_scales(bytes[i]);
    }
    if (cl == 0) {      // the tile's rows all get a scale, those past the matrix too: the tensor core reads 128 at a time
      uint8_t* sf = p.sf + fp8_sf_offset(r0, tile_c, p.kgroups);
#pragma unroll
      for (int i = 0; i < 8; ++i) sf[i * 16] = static_cast<uint8_t>(bytes[i >> 1] >> ((i & 1) * 16));
      if (p.ps != nullptr) {
        uint8_t* ps = p.ps + r0 * p.col_tiles + tile_c;
#pragma unroll
        for (int i = 0; i < 8; ++i, ps += p.col_tiles)
          if (i < nr) *ps = static_cast<uint8_t>(bytes[i >> 1] >> ((i & 1) * 16));
      }
    }
    if (c0 < p.q_ld) {
      uint8_t* out = p.q + r0 * p.q_ld + c0;
#pragma unroll
      for (int i = 0; i < 8; ++i, out += p.q_ld) {
        const uint2 codes = x.template row_codes<FMT>(i, inv[i >> 1]);
        if (i < nr) *reinterpret_cast<uint2*>(out) = codes;
      }
      if (odd) {
        out = p.q + r0 * p.q_ld + c0;
#pragma unroll 1
        for (int i = 0; i < nr; ++i, out += p.q_ld) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = x.at(i, j);
          fp8_fix_inf<FMT>(v, out, nc);
        }
      }
    }
  }
  if (COLS) {
    x.keep_packed();
    uint4 inv = make_uint4(0u, 0u, 0u, 0u);
    if (BLOCK) {
      inv.x = inv.y = inv.z = inv.w = fp8_inverse_scales(tile_bytes);
      const long long col = static_cast<long long>(tile_c) * QT + threadIdx.x;
      if (threadIdx.x < QT) {
        p.sft[fp8_sf_offset(col, tile_r, p.kgroups_t)] = static_cast<uint8_t>(tile_bytes);
        if (p.pst != nullptr && col < p.cols) p.pst[col * ((p.rows + QT - 1) / QT) + tile_r] = static_cast<uint8_t>(tile_bytes);
      }
    } else {
      __syncthreads();
      inv = *reinterpret_cast<const uint4*>(&s_inv[cl * 4]);
    }
    const uint32_t iw[4] = {inv.x, inv.y, inv.z, inv.w};
    // 8-byte unit rg of column 8 cl + j sits at unit rg ^ cl: the 16 lanes of a half-warp hit 16 different units
    uint8_t* mine = s_t + cl * 8 * QT + (rg ^ cl) * 8;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      uint2 codes[2];
      x.template column_codes<FMT>(j, iw[j >> 1], codes);
      *reinterpret_cast<uint2*>(mine + j * QT) = codes[0];
      *reinterpret_cast<uint2*>(mine + (j + 1) * QT) = codes[1];
    }
    if (odd) {
#pragma unroll 1
      for (int j = 0; j < 8; ++j) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = x.at(i, j);
        fp8_fix_inf<FMT>(v, mine + j * QT, 8);
      }
    }
    __syncthreads();
    const long long out_c = static_cast<long long>(tile_r) * QT + cl * 8;
    const long long left = p.cols - static_cast<long long>(tile_c) * QT;
    if (out_c < p.qt_ld) {
      uint8_t* out = p.qt + (static_cast<long long>(tile_c) * QT + rg) * p.qt_ld + out_c;
#pragma unroll
      for (int it = 0; it < QT / 16; ++it, out += 16 * p.qt_ld) {
        const int c = it * 16 + rg;                   // a half-warp writes the 128 bytes of one transposed row
        if (c < left)
          *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(s_t + c * QT + (cl ^ ((c >> 3) & 15)) * 8);
      }
    }
  }
  if (p.beside) wait_for_previous_kernel();
}

// Four CTAs an SM (64 registers, some spilled) where rows are written and there are eight tiles an SM or more, else three:
// both forms of 20480 x 3584 57.4 us with three, 53.2 with four; its rows 38.6 and 36.5; its transpose alone 40.2 and 42.1;
// both forms of 20480 x 1024 (1,280 tiles) 16.6 either way; of 4096 x 2048 (512 tiles) 8.2 and 8.9.
template <typename T, int FMT>
static void quant_launch(const QuantArgs& p, int mode, long long grid, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (grid > 8 * 148 && mode == 1)
      return launch_rows(fp8_quant_kernel<T, FMT, false, true, false, false, 4>, p, grid, Q_THREADS, s);
    if (grid > 8 * 148 && mode == 3)
      return launch_rows(fp8_quant_kernel<T, FMT, false, true, true, false, 4>, p, grid, Q_THREADS, s);
  }
  switch (mode) {
    case 1: launch_rows(fp8_quant_kernel<T, FMT, false, true, false, false>, p, grid, Q_THREADS, s); break;
    case 2: launch_rows(fp8_quant_kernel<T, FMT, false, false, true, false>, p, grid, Q_THREADS, s); break;
    case 3: launch_rows(fp8_quant_kernel<T, FMT, false, true, true, false>, p, grid, Q_THREADS, s); break;
    case 5: launch_rows(fp8_quant_kernel<T, FP8_E4M3, false, true, false, true>, p, grid, Q_THREADS, s); break;
    default: launch_rows(fp8_quant_kernel<T, FP8_E4M3, false, true, true, true>, p, grid, Q_THREADS, s); break;
  }
}

// ---------------------------------------------------------------------------------------------------
// h = x + resid (rounded to bf16, as a consumer reading it back would see it); y = h * rstd * (w_offset + w) in fp32,
// quantised without a bf16 rounding between.  Bound by HBM: 2 (x) + 2 (resid) read, 2 (h) + 1 + 1/128 written per
// element.  A row is held in registers from the read to the codes: TPR threads a row with NV vectors of 8 elements,
// 16 lanes to a block of 128, so its maximum is four shuffles.
// ---------------------------------------------------------------------------------------------------
struct NormQuantArgs {
  const __nv_bfloat16 *x, *resid, *w;
  __nv_bfloat16* h;
  uint8_t *q, *sf, *ps;       // ps: scale bytes in plain order; may be null
  float* rstd;
  long long rows, x_stride, r_stride, h_stride, q_ld;
  int D, kgroups, vec, beside;
  float eps, w_offset;
};

template <bool VEC>
__device__ __forceinline__ void store_raw8(__nv_bfloat16* p, const uint4& u, int n) {
  if (VEC) {
    if (n > 0) *reinterpret_cast<uint4*>(p) = u;
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(w[j >> 1] >> ((j & 1) * 16));
  }
}
__device__ __forceinline__ uint4 narrow8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

template <int TPR>
struct RowBlock {
  static constexpr int THREADS = TPR < 256 ? 256 : TPR;
  static constexpr int ROWS = THREADS / TPR;
};

template <int TPR, int NV, int FMT, bool VEC>
__global__ void __launch_bounds__(RowBlock<TPR>::THREADS)
fp8_norm_kernel(const NormQuantArgs p) {
  if (!p.beside) wait_for_previous_kernel();
  launch_dependents();
  constexpr int ROWS = RowBlock<TPR>::ROWS;
  __shared__ float s_part[ROWS][TPR / 32];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * ROWS + sub;
  const bool ok = row < p.rows;
  uint4 xr[NV], rr[NV], wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * 8, n = max(0, min(8, p.D - c));
    xr[i] = load_raw8<VEC>(p.x + row * p.x_stride + c, ok ? n : 0);
    rr[i] = load_raw8<VEC>(p.resid + row * p.r_stride + c, ok && p.resid != nullptr ? n : 0);
    wr[i] = load_raw8<VEC>(p.w + c, n);
  }
  float ss = 0.f, v[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    widen8(xr[i], v[i]);
    if (p.resid != nullptr) {
      const int c = (i * TPR + t) * 8, n = ok ? max(0, min(8, p.D - c)) : 0;
      float b[8];
      widen8(rr[i], b);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += b[j];
      const uint4 h = narrow8(v[i]);
      store_raw8<VEC>(p.h + row * p.h_stride + c, h, n);
      widen8(h, v[i]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
  }
  ss = warp_sum(ss);
  if (TPR > 32) {
    if (lane == 0) s_part[sub][t >> 5] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) ss += s_part[sub][i];
  }
  const float rstd = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(p.D)), p.eps));
  if (ok && t == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
  uint8_t* q = p.q + row * p.q_ld;
  uint8_t* sf = p.sf + fp8_sf_offset(row, 0, p.kgroups);
  uint8_t* ps = p.ps != nullptr ? p.ps + row * ((p.D + 127) / 128) : nullptr;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * 8, n = max(0, min(8, p.D - c));
    float g[8];
    widen8(wr[i], g);
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = VEC || j < n ? v[i][j] * rstd * (p.w_offset + g[j]) : 0.f;
    uint32_t m = fp8_max16(fp8_finite_max(v[i], &odd));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = fp8_scale_bytes<FMT>(m) & 0xFFu;
    if (ok && c < p.D && (t & 15) == 0) {
      sf[(c >> 9) * 512 + ((c >> 7) & 3)] = static_cast<uint8_t>(byte);
      if (ps != nullptr) ps[c >> 7] = static_cast<uint8_t>(byte);
    }
    if (ok && c < p.q_ld) {
      *reinterpret_cast<uint2*>(q + c) = fp8_pack8<FMT>(v[i], fp8_low(fp8_inverse_scales(byte)));
      if (odd) fp8_fix_inf<FMT>(v[i], q + c, n);
    }
  }
  if (p.beside) wait_for_previous_kernel();
}

template <int TPR, int NV>
static void norm_launch(const NormQuantArgs& p, int fmt, cudaStream_t s) {
  constexpr int THREADS = RowBlock<TPR>::THREADS;
  const unsigned grid = static_cast<unsigned>((p.rows + THREADS / TPR - 1) / (THREADS / TPR));
  if (p.vec) {
    if (fmt == FP8_E4M3) launch_rows(fp8_norm_kernel<TPR, NV, FP8_E4M3, true>, p, grid, THREADS, s);
    else launch_rows(fp8_norm_kernel<TPR, NV, FP8_E5M2, true>, p, grid, THREADS, s);
  } else {
    if (fmt == FP8_E4M3) launch_rows(fp8_norm_kernel<TPR, NV, FP8_E4M3, false>, p, grid, THREADS, s);
    else launch_rows(fp8_norm_kernel<TPR, NV, FP8_E5M2, false>, p, grid, THREADS, s);
  }
}

// ---------------------------------------------------------------------------------------------------
// Backward of the norm, dn (fp32) = gradient of its output:  g = dn * (w_offset + w), xh = h * rstd,
//   dx = rstd * (g - xh * mean(g * xh)) + dh,        dw = sum over rows of dn * xh.
// dn comes straight from the product's fp32 sums: rounding it to bf16 between the two would put a second rounding, as
// large as the result's own, into every gradient.  Bound by HBM: 4 (dn) + 2 (h) + 2 (dh) read, 2 written per element.
// Every CTA walks rows at a stride of the grid; a thread keeps a row's values packed as they were read and its share
// of dw in registers.  The shares are summed in a fixed order by a second kernel, so dw is the same from run to run.
// ---------------------------------------------------------------------------------------------------
struct NormBwdArgs {
  const float* dn;
  const __nv_bfloat16 *h, *w, *dh;
  const float* rstd;
  __nv_bfloat16* dx;
  float* part;       // [grid, D]
  long long rows, dn_stride, h_stride, dh_stride;
  int D, vec;
  float w_offset;
};

template <bool VEC>
__device__ __forceinline__ void load_f32x8(const float* p, int n, float (&v)[8]) {
  if (VEC) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (n > 0) {
      a = __ldg(reinterpret_cast<const float4*>(p));
      b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? p[j] : 0.f;
  }
}

// The next row's vectors are loaded before this row's are used: a CTA waits for its row's sum in between, and without
// them the SM had loads in flight for half of the time ([40960, 1024]: 93 us, 65 % of HBM).  TPR = 1024 has no registers
// for that.
template <int TPR, int NV>
struct NormBwd {
  static constexpr bool AHEAD = TPR < 1024;
  static constexpr int MIN_CTAS = TPR >= 512 ? 1 : NV == 2 ? 2 : 3;
};
template <int NV>
struct NormBwdRow {
  uint4 h[NV], dh[NV];
  float dn[NV][8];
  float rstd;
};

template <int TPR, int NV, bool VEC>
__device__ __forceinline__ void norm_bwd_load(const NormBwdArgs& p, long long row, int t, NormBwdRow<NV>& r) {
  const bool ok = row < p.rows;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * 8, n = ok ? max(0, min(8, p.D - c)) : 0;
    r.h[i] = load_raw8<VEC>(p.h + row * p.h_stride + c, n);
    load_f32x8<VEC>(p.dn + row * p.dn_stride + c, n, r.dn[i]);
    r.dh[i] = load_raw8<VEC>(p.dh + row * p.dh_stride + c, p.dh != nullptr ? n : 0);
  }
  r.rstd = ok ? p.rstd[row] : 0.f;
}

template <int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(RowBlock<TPR>::THREADS, NormBwd<TPR, NV>::MIN_CTAS)
fp8_norm_bwd_kernel(const NormBwdArgs p) {
  constexpr int ROWS = RowBlock<TPR>::ROWS;
  __shared__ float s_part[2][ROWS][TPR / 32];
  __shared__ float s_dw[ROWS > 1 ? TPR * NV * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, lane = threadIdx.x & 31;
  float acc[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  uint4 wr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) wr[i] = load_raw8<VEC>(p.w + (i * TPR + t) * 8, max(0, min(8, p.D - (i * TPR + t) * 8)));
  int flip = 0;
  const long long step = static_cast<long long>(gridDim.x) * ROWS;
  NormBwdRow<NV> cur, next;
  norm_bwd_load<TPR, NV, VEC>(p, static_cast<long long>(blockIdx.x) * ROWS + sub, t, cur);
  // the trip count is the block's, not the row group's: TPR > 32 synchronises inside
  for (long long r0 = static_cast<long long>(blockIdx.x) * ROWS; r0 < p.rows; r0 += step) {
    const long long row = r0 + sub;
    const bool ok = row < p.rows;
    if (NormBwd<TPR, NV>::AHEAD) norm_bwd_load<TPR, NV, VEC>(p, row + step, t, next);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float xh[8], w8[8];
      widen8(cur.h[i], xh);
      widen8(wr[i], w8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = xh[j] * cur.rstd;
        acc[i][j] += cur.dn[i][j] * x;
        cur.dn[i][j] *= p.w_offset + w8[j];
        dot += cur.dn[i][j] * x;             // both are zero outside the row
      }
    }
    dot = warp_sum(dot);
    if (TPR > 32) {
      if (lane == 0) s_part[flip][sub][t >> 5] = dot;
      __syncthreads();                   // the other buffer's readers are all past the barrier before this one
      dot = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 32; ++i) dot += s_part[flip][sub][i];
      flip ^= 1;
    }
    dot *= cur.rstd / p.D;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * 8, n = ok ? max(0, min(8, p.D - c)) : 0;
      float xh[8], d8[8];
      widen8(cur.h[i], xh);
      widen8(cur.dh[i], d8);
#pragma unroll
      for (int j = 0; j < 8; ++j) d8[j] += cur.rstd * (cur.dn[i][j] - xh[j] * dot);
      store_raw8<VEC>(p.dx + row * p.D + c, narrow8(d8), n);
    }
    if (NormBwd<TPR, NV>::AHEAD) cur = next;
    else norm_bwd_load<TPR, NV, VEC>(p, row + step, t, cur);
  }
  if (p.part == nullptr) return;
  float* part = p.part + static_cast<long long>(blockIdx.x) * p.D;
  // the row groups add their shares one after the other, in the same order every time
  for (int g = 0; g < ROWS; ++g) {
    if (sub == g) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = (i * TPR + t) * 8 + j;
          const float v = g > 0 ? s_dw[ROWS > 1 ? (i * 8 + j) * TPR + t : 0] + acc[i][j] : acc[i][j];
          if (g < ROWS - 1) s_dw[ROWS > 1 ? (i * 8 + j) * TPR + t : 0] = v;
          else if (c < p.D) part[c] = v;
        }
    }
    if (ROWS > 1) __syncthreads();
  }
}

// dw[c] = sum over the parts in a fixed order: 32 groups of consecutive parts, then the groups; fp32 +=, or bf16
__global__ void __launch_bounds__(1024)
fp8_norm_dw_kernel(const float* __restrict__ part, int parts, int D, float* __restrict__ acc,
                   __nv_bfloat16* __restrict__ out) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  const int per = (parts + 31) / 32;
  float sum = 0.f;
  if (c < D)
    for (int i = g * per; i < min(parts, (g + 1) * per); ++i) sum += part[static_cast<long long>(i) * D + c];
  s[g][threadIdx.x & 31] = sum;
  __syncthreads();
  if (g == 0 && c < D) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) total += s[i][threadIdx.x & 31];
    if (acc != nullptr) acc[c] += total;
    else out[c] = __float2bfloat16_rn(total);
  }
}

constexpr int NORM_BWD_MAX_PARTS = 444;   // 148 SMs with three CTAs each

template <int TPR, int NV>
static int norm_bwd_launch(const NormBwdArgs& p, cudaStream_t s) {
  constexpr int THREADS = RowBlock<TPR>::THREADS;
  const long long want = (p.rows + THREADS / TPR - 1) / (THREADS / TPR);
  const int resident = 148 * NormBwd<TPR, NV>::MIN_CTAS;
  const int grid = static_cast<int>(want < resident ? want : resident);
  if (p.vec) fp8_norm_bwd_kernel<TPR, NV, true><<<grid, THREADS, 0, s>>>(p);
  else fp8_norm_bwd_kernel<TPR, NV, false><<<grid, THREADS, 0, s>>>(p);
  return grid;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace cvb

using namespace cvb;

// ps, pst (may be null): the scale bytes once more, in plain order, for other programs to read
// mode: 1 row form, 2 transposed form, 3 both, 5 row form with 128 x 128 blocks, 7 both with 128 x 128 blocks
extern "C" int cvb_fp8_quantize(const void* x, int x_fp32, long long rows, long long cols, long long x_stride, int fmt,
                                int mode, void* q, void* sf, void* ps, long long q_ld, void* qt, void* sft, void* pst,
                                long long qt_ld, const float* rstd, const void* w, float w_offset, int beside, void* stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((fmt != FP8_E4M3 && fmt != FP8_E5M2) || (mode != 1 && mode != 2 && mode != 3 && mode != 5 && mode != 7)) return -1;
  if (mode > 3 && fmt != FP8_E4M3) return -1;
  if (((mode & 1) && (!q || !sf || !aligned16(q) || q_ld % 16 || q_ld < cols)) ||
      ((mode & 2) && (!qt || !sft || !aligned16(qt) || qt_ld % 16 || qt_ld < rows)))
    return -2;
  if ((rstd != nullptr) != (w != nullptr) || (rstd != nullptr && (x_fp32 || mode != 2 || fmt != FP8_E4M3))) return -3;
  const long long row_tiles = (rows + QT - 1) / QT, col_tiles = (cols + QT - 1) / QT;
  if (row_tiles * col_tiles > 0x7fffffffll) return -4;
  const int elem = x_fp32 ? 4 : 2;
  QuantArgs p = {};
  p.x = x;
  p.rows = rows, p.cols = cols, p.x_stride = x_stride;
  p.vec = aligned16(x) && (x_stride * elem) % 16 == 0;
  p.q = static_cast<uint8_t*>(q), p.sf = static_cast<uint8_t*>(sf), p.q_ld = q_ld;
  p.kgroups = static_cast<int>((col_tiles + 3) / 4);
  p.ps = static_cast<uint8_t*>(ps), p.pst = static_cast<uint8_t*>(pst);
  p.qt = static_cast<uint8_t*>(qt), p.sft = static_cast<uint8_t*>(sft), p.qt_ld = qt_ld;
  p.kgroups_t = static_cast<int>((row_tiles + 3) / 4);
  p.col_tiles = static_cast<int>(col_tiles);
  p.rstd = rstd, p.w = static_cast<const __nv_bfloat16*>(w), p.w_offset = w_offset, p.beside = beside;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long grid = row_tiles * col_tiles;
  if (rstd != nullptr) {     // the transposed form of a norm's result: what a weight gradient reads
    launch_rows(fp8_quant_kernel<__nv_bfloat16, FP8_E4M3, true, false, true, false>, p, grid, Q_THREADS, s);
  } else if (x_fp32) {
    if (fmt == FP8_E4M3) quant_launch<float, FP8_E4M3>(p, mode, grid, s);
    else quant_launch<float, FP8_E5M2>(p, mode, grid, s);
  } else {
    if (fmt == FP8_E4M3) quant_launch<__nv_bfloat16, FP8_E4M3>(p, mode, grid, s);
    else quant_launch<__nv_bfloat16, FP8_E5M2>(p, mode, grid, s);
  }
  return static_cast<int>(cudaGetLastError());
}

extern "C" int cvb_fp8_add_rmsnorm(const void* x, long long x_stride, const void* resid, long long r_stride,
                                   const void* w, void* h, void* q, void* sf, void* ps, long long q_ld, float* rstd,
                                   long long rows, int D, int fmt, float eps, float w_offset, int beside,
                                   void* stream) {
  if (rows <= 0 || D <= 0) return 0;
  if (fmt != FP8_E4M3 && fmt != FP8_E5M2) return -1;
  if (!aligned16(q) || q_ld % 16 || q_ld < D || (resid != nullptr) != (h != nullptr)) return -2;
  if (D > 16384 || rows > 0x7fffffffll) return -3;
  NormQuantArgs p = {};
  p.x = static_cast<const __nv_bfloat16*>(x), p.resid = static_cast<const __nv_bfloat16*>(resid);
  p.w = static_cast<const __nv_bfloat16*>(w), p.h = static_cast<__nv_bfloat16*>(h);
  p.q = static_cast<uint8_t*>(q), p.sf = static_cast<uint8_t*>(sf), p.ps = static_cast<uint8_t*>(ps), p.rstd = rstd;
  p.rows = rows, p.x_stride = x_stride, p.r_stride = r_stride, p.h_stride = D, p.q_ld = q_ld;
  p.D = D, p.kgroups = ((D + 127) / 128 + 3) / 4;
  p.vec = aligned16(x) && aligned16(resid) && aligned16(w) && aligned16(h) && x_stride % 8 == 0 && r_stride % 8 == 0 &&
          D % 8 == 0;
  p.eps = eps, p.w_offset = w_offset, p.beside = beside;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // the fewest threads that hold a row with at most four vectors each
  if (D <= 256) norm_launch<32, 1>(p, fmt, s);
  else if (D <= 512) norm_launch<32, 2>(p, fmt, s);
  else if (D <= 1024) norm_launch<32, 4>(p, fmt, s);
  else if (D <= 2048) norm_launch<128, 2>(p, fmt, s);
  else if (D <= 4096) norm_launch<128, 4>(p, fmt, s);
  else if (D <= 8192) norm_launch<256, 4>(p, fmt, s);
  else norm_launch<512, 4>(p, fmt, s);
  return static_cast<int>(cudaGetLastError());
}

// rows of the workspace [parts, D] that cvb_fp8_norm_bwd may fill
extern "C" int cvb_fp8_norm_bwd_parts(void) { return NORM_BWD_MAX_PARTS; }

// dw_acc (fp32, +=) or dw (bf16); both null: no weight gradient
extern "C" int cvb_fp8_norm_bwd(const float* dn, long long dn_stride, const void* h, long long h_stride, const void* w,
                                const float* rstd, const void* dh, long long dh_stride, void* dx, float* part,
                                float* dw_acc, void* dw, long long rows, int D, float w_offset, void* stream) {
  if (rows <= 0 || D <= 0) return 0;
  if (D > 16384) return -3;
  if ((dw_acc != nullptr || dw != nullptr) && part == nullptr) return -2;
  NormBwdArgs p = {};
  p.dn = dn, p.h = static_cast<const __nv_bfloat16*>(h);
  p.w = static_cast<const __nv_bfloat16*>(w), p.dh = static_cast<const __nv_bfloat16*>(dh);
  p.rstd = rstd, p.dx = static_cast<__nv_bfloat16*>(dx);
  p.part = dw_acc != nullptr || dw != nullptr ? part : nullptr;
  p.rows = rows, p.dn_stride = dn_stride, p.h_stride = h_stride, p.dh_stride = dh_stride, p.D = D;
  p.vec = aligned16(dn) && aligned16(h) && aligned16(w) && aligned16(dh) && aligned16(dx) && dn_stride % 4 == 0 &&
          h_stride % 8 == 0 && dh_stride % 8 == 0 && D % 8 == 0;
  p.w_offset = w_offset;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int grid;
  if (D <= 256) grid = norm_bwd_launch<32, 1>(p, s);
  else if (D <= 512) grid = norm_bwd_launch<64, 1>(p, s);
  else if (D <= 1024) grid = norm_bwd_launch<128, 1>(p, s);
  else if (D <= 2048) grid = norm_bwd_launch<256, 1>(p, s);
  else if (D <= 4096) grid = norm_bwd_launch<256, 2>(p, s);
  else if (D <= 8192) grid = norm_bwd_launch<512, 2>(p, s);
  else grid = norm_bwd_launch<1024, 2>(p, s);
  if (p.part != nullptr)
    fp8_norm_dw_kernel<<<(D + 31) / 32, 1024, 0, s>>>(part, grid, D, dw_acc, static_cast<__nv_bfloat16*>(dw));
  return static_cast<int>(cudaGetLastError());
}
