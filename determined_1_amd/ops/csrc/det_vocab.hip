// det_vocab: losses of a language model's last layer over a vocabulary of V words, without its logits.
//
// A row n (token) has a hidden state h_n [D]; word v has a weight row w_v [D] and a bias b_v.
//     z_nv = (h_n . w_v + b_v) / T        lse_n = log sum_v exp z_nv        p_nv = exp(z_nv - lse_n)
// Both losses compare p_n with a sparse distribution s_n over K words (index a_nk, share s_nk):
//     cross entropy  K = 1, s = 1 - eps, T = 1, and eps / V on every word (label smoothing):
//                    loss_n = lse_n - (1 - eps) z_n,target - eps / V sum_v z_nv
//     distillation   s_n = softmax of the teacher's K top logits / T, in the same units:
//                    loss_n = T^2 sum_k s_nk (log s_nk - z_n,a_nk + lse_n)
// and have one derivative, G_nv = c_n (p_nv - eps / V - sum_k s_nk [a_nk = v]), from which
//     dh_n = sum_v G_nv w_v        dw_v = sum_n G_nv h_n        db_v = sum_n G_nv.
//
// Forward: one product [rows x D] . [D x V] whose epilogue reduces each tile of logits to a maximum and a
// sum of exponentials per row (and hands out the target's logit); a joining pass per row, which for lists
// adds the K listed logits, dot products of their own.  Backward: the vocabulary is walked in chunks; per
// chunk G is written to a workspace, and two more products read it.  G comes from the tile's exponentials,
// which the forward held (hold_bits; with smoothing and for fp32 in fp32) as far as the caller's bound goes (2 GiB
// unless it says otherwise), and past that from the product once more, in its epilogue.  What bounds it, 8192 x 4096
// x 128000 bf16 in 22.3 ms: the matrix units, 1.24 PFLOP/s over the three products (logits 6.8 ms, G w 6.8, G^T h
// 7.2; G from 2 GB of exponentials 0.8, where the product again takes 6.7); for few rows the reads of w (one row
// against 128000 x 4096: 6.0 TB/s).
//
// Rows without a target are dropped before the products (an ordered list of the kept ones, made on the
// device; tiles past its end return), so a masked-language-model step with 15 % targets costs 15 %.
//
// G is held in the operands' 16 bits, which the matrix units take: each entry is off by at most half a step
// (bf16 2^-8), at random, so gradients of many rows are off by about as much as their own rounding once more
// (bf16 2048 x 2048 x 32000: 0.0023 against 0.0017 of their size).  With few rows one entry of one row can
// decide: there G is two 16-bit rows each, the second what the first one's rounding took, which only fills
// what is left of a tile.  A bias gradient comes from G before its rounding.  Everything else is fp32.
//
// fp32 operands become two fp16 planes each, x s = hi + lo with s a power of two that puts the largest finite
// magnitude at 2^14..2^15: of each row of h in the logits, of all kept rows in G^T h, of all words in w, those that a
// bias of -inf takes out not among them.  A product is hi hi + hi lo + lo hi in fp32 accumulators: each operand is
// held to 2^-23 of itself, or 2^-39 of that largest magnitude where that is more (entries of w, or of h for dw, more
// than 2^16 below it lose bits that an fp32 product keeps), and the dropped lo lo is below 2^-22 of its product, the
// size of one fp32 rounding, at a third of the matrix units' 16-bit rate instead of the sixteenth that their fp32
// instructions have (2240 x 850 x 10000: off by 5e-7 of the gradients' size, an fp32 product by 1.8e-6).
#include <hip/hip_runtime.h>

#include <atomic>
#include <cstdint>
#include <type_traits>

namespace {

typedef unsigned short u16;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) u16 us8;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };  // element types, as in _lib.py

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_huge_valf();

template <int DT> struct Elem;
template <> struct Elem<kF32> { typedef float type; };
template <> struct Elem<kBF16> { typedef u16 type; };
template <> struct Elem<kF16> { typedef u16 type; };

__device__ __forceinline__ float bf2f(u16 u) { return __uint_as_float(static_cast<uint32_t>(u) << 16); }
__device__ __forceinline__ u16 f2bf(float f) { return __builtin_bit_cast(u16, static_cast<__bf16>(f)); }
__device__ __forceinline__ float h2f(u16 u) { return static_cast<float>(__builtin_bit_cast(_Float16, u)); }
__device__ __forceinline__ u16 f2h(float f) { return __builtin_bit_cast(u16, static_cast<_Float16>(f)); }

// The value as an fp32 register.  Without it the compiler may round a product to fp16 in one instruction for
// the upper plane and from fp32 for the lower one: at a tie the planes then miss each other by a step.
__device__ __forceinline__ float settled(float v) {
  asm("" : "+v"(v));
  return v;
}

template <int DT>
__device__ __forceinline__ float to_f(typename Elem<DT>::type v) {
  if constexpr (DT == kF32) return v;
  else if constexpr (DT == kBF16) return bf2f(v);
  else return h2f(v);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::type from_f(float f) {
  if constexpr (DT == kF32) return f;
  else if constexpr (DT == kBF16) return f2bf(f);
  else return f2h(f);
}
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dt) {
  return dt == kF32 ? static_cast<const float*>(p)[i] : dt == kBF16 ? bf2f(static_cast<const u16*>(p)[i])
                                                                    : h2f(static_cast<const u16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dt, float f) {
  if (dt == kF32) static_cast<float*>(p)[i] = f;
  else static_cast<u16*>(p)[i] = dt == kBF16 ? f2bf(f) : f2h(f);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// The running maximum m and sum s of 2^(c (z - m)), c = log2(e) / T: (m, s) + (m2, s2).  A maximum of -inf
// stands for nothing yet.  Maximum and sum stay apart up to the end (no m + log s): logits masked with the
// type's lowest value would absorb the logarithm, and times log2(e) they would be out of range.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float c) {
  const float hi = fmaxf(m, m2);
  const float ref = hi == kNegInf ? 0.f : hi;
  s = s * exp2_((m - ref) * c) + s2 * exp2_((m2 - ref) * c);
  m = hi;
}
__device__ __forceinline__ void join_lanes(float& m, float& s, int width, float c) {
  for (int o = 1; o < width; o <<= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
    join(m, s, m2, s2, c);
  }
}
__device__ __forceinline__ float sum_lanes(float v) {
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float max_lanes(float v) {
  for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// the exponent of the power of two that brings a tensor's largest finite magnitude (its bits) to [2^14, 2^15): from
// -113 to 141, so that the power itself may be out of range and is applied by ldexp
__device__ __forceinline__ int scale_exp(uint32_t bits) { return bits == 0 ? 0 : 141 - static_cast<int>(bits >> 23); }
__device__ __forceinline__ float times_pow2(float v, int e) { return __builtin_ldexpf(v, e); }

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

constexpr int kGExp = 14;  // fp16 G is held times 2^14: |G| <= 1 stays below 65504, its smallest step is 2^-38

// ------------------------------------------------------------------------------------------------
// Rows: the ordered list of the rows that count, by one block (its order is what makes it one: 7 us for
// 4608 rows, 14 for 8192).  info[0] = how many, info[1], info[2] = the largest
// finite magnitudes (as bits) of the hidden states and the weights, cleared here for absmax_kernel.
// ------------------------------------------------------------------------------------------------
struct RowArgs {
  const void* target;   // cross entropy: [N] words, else null
  const void* index;    // distillation: [N, K] words (< 0: no entry)
  const void* teacher;  // [N, K] logits (-inf: no entry)
  uint8_t* flag;        // [N], distillation
  int* info;
  int* list;   // [N] the kept rows, in order
  int* pos;    // [N] a row's place in the list, or -1
  int* words;  // [kept] cross entropy: the target, or -1 outside the vocabulary
  float* each; // [N] losses to clear for rows that do not count, or null
  int64_t ignore, index_ld, teacher_ld;
  int N, K, V, wide, teacher_dt;
};

__global__ void __launch_bounds__(256) list_flags_kernel(RowArgs a) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= a.N) return;
  bool any = false;
  for (int k = lane; k < a.K; k += 64)
    any |= load_index(a.index, n * a.index_ld + k, a.wide) >= 0 && load_any(a.teacher, n * a.teacher_ld + k, a.teacher_dt) != kNegInf;
  const uint64_t votes = __ballot(any);
  if (lane == 0) a.flag[n] = votes != 0;
}

// one block; eight neighbouring rows a thread, whose targets are read together
__global__ void __launch_bounds__(1024) rows_kernel(RowArgs a) {
  __shared__ int wave_n[16];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int done = 0;  // kept rows of earlier rounds
  for (int n0 = 0; n0 < a.N; n0 += 8192) {
    const int first = n0 + tid * 8;
    int64_t word[8];
    unsigned keep = 0;
    const bool eight = a.target != nullptr && a.wide && first + 8 <= a.N && (reinterpret_cast<uintptr_t>(a.target) & 15) == 0;
    if (eight) __builtin_memcpy(word, __builtin_assume_aligned(static_cast<const int64_t*>(a.target) + first, 16), sizeof(word));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (eight) {
        keep |= (word[e] != a.ignore ? 1u : 0u) << e;
        continue;
      }
      word[e] = 0;
      if (first + e < a.N) {
        if (a.target != nullptr) {
          word[e] = load_index(a.target, first + e, a.wide);
          keep |= (word[e] != a.ignore ? 1u : 0u) << e;
        } else {
          keep |= (a.flag[first + e] != 0 ? 1u : 0u) << e;
        }
      }
    }
    const int mine = __popc(keep);
    int upto = mine;  // with the lanes below
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
    if (lane == 63) wave_n[w] = upto;
    __syncthreads();
    int at = done + upto - mine;
    for (int i = 0; i < 16; ++i) {
      if (i < w) at += wave_n[i];
      done += wave_n[i];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int n = first + e;
      if (n >= a.N) continue;
      const bool k = (keep >> e) & 1;
      a.pos[n] = k ? at : -1;
      if (k) {
        a.list[at] = n;
        if (a.target != nullptr) a.words[at] = word[e] >= 0 && word[e] < a.V ? static_cast<int>(word[e]) : -1;
        ++at;
      } else if (a.each != nullptr) {
        a.each[n] = 0.f;
      }
    }
    __syncthreads();
  }
  if (tid == 0) {
    a.info[0] = done;
    a.info[1] = 0;
    a.info[2] = 0;
  }
}

// The largest finite magnitudes of the hidden states and the weights (fp32), as bits: blocks below
// x_blocks go over x, its kept rows alone (what an ignored one holds must not decide their scale), and leave each
// row's as well; of the weights, words that a bias of -inf takes out do not count either.  One atomic a block (eight
// thousand, one a wave, took 65 us of a 75 us launch); a maximum does not depend on their order.  Bound by the
// read of w (333 x 768 against 30522 words: 94 MB in 30 us, 3.1 TB/s).
struct Matrix {
  const float* p;
  int64_t ld;
  int rows, cols;
  const int *list, *count;  // the rows that count, and how many (null: all)
  int* each;                // their magnitudes, with a list
  const void* bias;         // the weights': null or [rows]
  int bias_dt;
};

// a word that its bias takes out: z is -inf whatever its row of the weights holds
__device__ __forceinline__ bool masked(const void* bias, int64_t word, int dt) { return bias != nullptr && load_any(bias, word, dt) == kNegInf; }

// four values from any address (16-byte loads need no alignment here), zeros past the row's end
__device__ __forceinline__ f32x4 load4(const float* p, int there) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (there >= 4) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e) v[e] = e < there ? p[e] : 0.f;
  }
  return v;
}

__global__ void __launch_bounds__(256) absmax_kernel(Matrix x, Matrix w, int x_blocks, int* info) {
  __shared__ uint32_t red[4];
  const bool isx = blockIdx.x < static_cast<unsigned>(x_blocks);
  const Matrix a = isx ? x : w;
  const int64_t block = isx ? blockIdx.x : blockIdx.x - x_blocks, blocks = isx ? x_blocks : gridDim.x - x_blocks;
  uint32_t m = 0;
  auto take = [&](float f) {
    const uint32_t b = __float_as_uint(f) & 0x7FFFFFFFu;
    if (b < 0x7F800000u && b > m) m = b;
  };
  auto most = [](uint32_t v) {
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_xor(v, o, 64);
      v = u > v ? u : v;
    }
    return v;
  };
  const int64_t all = static_cast<int64_t>(a.rows) * a.cols;
  if (a.list == nullptr && a.bias == nullptr && a.ld == a.cols && (reinterpret_cast<uintptr_t>(a.p) & 15) == 0) {
#pragma unroll 4
    for (int64_t i = block * 256 + threadIdx.x; i < all / 4; i += blocks * 256) {
      const f32x4 v = reinterpret_cast<const f32x4*>(a.p)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) take(v[e]);
    }
    if (block == 0 && threadIdx.x < (all & 3)) take(a.p[all - 1 - threadIdx.x]);
  } else if (a.list == nullptr) {  // four rows of a block on their way at a time
    for (int64_t r0 = block * 4; r0 < a.rows; r0 += blocks * 4) {
      bool there[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) there[q] = r0 + q < a.rows && !masked(a.bias, r0 + q, a.bias_dt);
      for (int c = threadIdx.x * 4; c < a.cols; c += 1024) {
        f32x4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = there[q] ? load4(a.p + (r0 + q) * a.ld + c, a.cols - c) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 4; ++e) take(v[q][e]);
      }
    }
  } else {  // a row a wave
    const int rows = *a.count;
    uint32_t all_rows = 0;
    for (int64_t r = block * 4 + (threadIdx.x >> 6); r < rows; r += blocks * 4) {
      const float* p = a.p + a.list[r] * a.ld;
      m = 0;
#pragma unroll 4
      for (int c = (threadIdx.x & 63) * 4; c < a.cols; c += 256) {
        const f32x4 v = load4(p + c, a.cols - c);
#pragma unroll
        for (int e = 0; e < 4; ++e) take(v[e]);
      }
      m = most(m);
      if ((threadIdx.x & 63) == 0) a.each[r] = static_cast<int>(m);
      all_rows = m > all_rows ? m : all_rows;
    }
    m = all_rows;
  }
  m = most(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i) m = red[i] > m ? red[i] : m;
    atomicMax(reinterpret_cast<unsigned int*>(info + (isx ? 1 : 2)), m);
  }
}

// ------------------------------------------------------------------------------------------------
// Operands of the products: 16-bit rows, 16-byte aligned, columns past the width zero.  Copies the
// rows of `list` (or all), and splits fp32 into two fp16 planes.  Bound by memory: 128000 x 4096 fp32 in
// 0.85 ms, 4.9 TB/s.  The hidden states always (their kept rows move together), weights only if they are
// fp32, of a width or a row distance that 16 bytes do not divide, or misaligned.  DT kBF16 copies any 16-bit type as
// bits; kF16 is for rows times a power of two.
// ------------------------------------------------------------------------------------------------
struct PackArgs {
  const void* src;
  int64_t src_ld;
  const int* list;   // null: rows as they are
  const int* count;  // null: `rows`
  const int* absmax; // fp32: the largest magnitude that the scale is for,
  const int* each;   // or each row's
  u16* dst;
  int64_t plane;     // elements between the planes
  int rows, cols, ld;  // ld % 8 == 0
  int twice;         // the rows once more behind the last one
  const int* row_e;  // rows times 2^row_e, or null
  const void* bias;  // words (fp32) that it takes out are zeros, or null
  int bias_dt;
};

// eight elements from any address (16-byte loads need no alignment here), zeros past the row's end
template <class T>
__device__ __forceinline__ void load8(const T* p, int there, T (&v)[8]) {
  if (there >= 8) {
    __builtin_memcpy(v, p, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < there ? p[e] : T(0);
  }
}

template <int DT>
__global__ void __launch_bounds__(256) pack_kernel(PackArgs a) {
  typedef typename Elem<DT>::type T;
  const int rows = a.count != nullptr ? *a.count : a.rows;
  const int chunks = a.ld >> 3;
  // a thread per eight columns, whatever the width
  const int64_t all = static_cast<int64_t>(rows) * chunks, step = gridDim.x * 256ll;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += step) {
    const int r = static_cast<int>(i / chunks), c = static_cast<int>(i - static_cast<int64_t>(r) * chunks) * 8;
    const int more = a.row_e != nullptr ? a.row_e[r] : 0;
    const int64_t from = static_cast<int64_t>(a.list != nullptr ? a.list[r] : r) * a.src_ld;
    const int scale = DT == kF32 ? scale_exp(static_cast<uint32_t>(a.each != nullptr ? a.each[r] : *a.absmax)) : 0;
    T v[8];
    load8(static_cast<const T*>(a.src) + from + c, DT == kF32 && masked(a.bias, r, a.bias_dt) ? 0 : a.cols - c, v);
    us8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == kF32) {
        const float x = times_pow2(v[e], scale + more);
        hi[e] = f2h(x);
        lo[e] = f2h(x - h2f(hi[e]));
      } else if constexpr (DT == kF16) {
        hi[e] = f2h(times_pow2(h2f(v[e]), more));
      } else {
        hi[e] = v[e];
      }
    }
    u16* d = a.dst + static_cast<int64_t>(r) * a.ld + c;
    *reinterpret_cast<us8*>(d) = hi;
    if constexpr (DT == kF32) *reinterpret_cast<us8*>(d + a.plane) = lo;
    else if (a.twice) *reinterpret_cast<us8*>(d + static_cast<int64_t>(rows) * a.ld) = hi;
  }
}

// ------------------------------------------------------------------------------------------------
// The products.  C tile 256 x 256, 8 waves as 2 (rows) x 4 (columns) of 128 x 64, v_mfma 16x16x32.
// An operand lies with its k contiguous ("row": element (i, k) at i * ld + k) or strided ("col":
// (i, k) at k * ld + i, read back from LDS transposed).  LDS holds 8 KiB images of 128 rows (or columns)
// by 32 k, in stages of both operands' 256 and, for a split fp32 operand, both planes.
// Bound by what feeds the matrix units: a stage of 64 k is 2048 cycles of them and of fragment reads (192 KiB)
// and fetches (64 KiB) through LDS nearly as many, which share its port; 0.93 us a stage with neither, 1.1 with
// one of them, 1.3 with both, 1.45 with data that makes the clock drop.
// Everything outside an operand's extents is fetched out of the buffer's range, which gives zeros.
// ------------------------------------------------------------------------------------------------
// A gradient's scale: G is held in [-1, 1] 2^k, row weights divided by the largest one's magnitude.
struct Alpha {
  const float* p;   // the loss's derivative, or the largest one of a row's
  const int* info;
  float scale;      // T / 2^k
  int mean;
  __device__ __forceinline__ float operator()() const {
    const int count = info[0];
    if (count == 0) return 0.f;  // no row's gradient, whatever the derivative is
    return *p * scale / (mean ? static_cast<float>(count) : 1.f);
  }
};

struct Operand {
  const u16* p;
  int64_t plane, ld;
};

enum { kStats, kGrad, kPartial, kOut };

struct GemmArgs {
  Operand A, B;
  const int* m_dyn;  // rows of A that count (null: M)
  const int* k_dyn;  // length of the sum (null: K)
  int twice;         // rows of G are two: kGrad writes both, kPartial and kOut read twice as many as m_dyn or k_dyn says
  int M, N, K;
  int least;                // kPartial: the shortest piece
  int chunk;                // kPartial of words: the longest K of the pass, which the splits are made for
  int cut;                  // whether the last round's tiles may be cut in two
  // what the scales of fp32 operands are made of: kStats, kGrad: each row's of A, info[2] for B; kOut: B's
  const int *info, *bits;
  // kStats, kGrad: z = acc / scales + bias, c = log2(e) / T
  const void* bias;
  int bias_dt;
  float c;
  float2* part;   // kStats [M][parts], 128 columns each: maximum and sum
  // kStats: the first `held` words' exponentials below the tile's maximum (null: none), and the maxima
  void* E;        // [M][held], 11-bit numbers, or fp32 if exact
  int exact;
  float* tops;    // [M][held / 128]
  int held;       // (a multiple of 256)
  float* part_z;  // sum of z / V, or null
  float inv_v;
  int parts;
  // kGrad: p = 2^(c (z - top) - log2 sum)
  const float *top, *log_s;  // [M]
  const float* row_w;        // [M] (null: g_scale for each)
  const int* row_e;          // [M] row_w's rows are to be taken times 2^row_e (null: as they are)
  float g_scale;
  float smooth_v;      // eps / V
  float* colsum;       // [tiles of M][ldg] G's column sums, or null
  // kStats, kGrad for one target a row: the words (null for lists), the word of column 0, the target's
  // logit (kStats writes it), its share
  const int* words;
  int v0;
  float* picked;
  float share;
  u16* G;              // [M][ldg]
  int64_t g_plane;
  int ldg;
  // kPartial: out[split][M][ldo] fp32 (ldo % 4 == 0), added to what is there if `add`
  float* out32;
  int64_t ldo;
  int add;
  // kOut: out[m][n] of the operands' type (fp32 if split), times *alpha and the scale of B
  void* out;
  Alpha alpha;
};

// Few tiles: their sum (over a chunk's words for G w, over the kept rows for G^T h, over D for logits) is cut
// until a block runs on every CU (one fills a CU), no piece under `least` long.  The length of a piece, a
// multiple of 64.
constexpr int kPiece = 512, kLogitPiece = 256;
__host__ __device__ inline int split_length(int tiles, int span, int least) {
  int splits = tiles < 256 ? 256 / tiles : 1;
  const int most = span / least > 1 ? span / least : 1;
  if (splits > most) splits = most;
  return ((span + splits - 1) / splits + 63) / 64 * 64;
}

constexpr int kTile = 256, kThreads = 512;
constexpr int kHalf = 16384, kStage = 4 * kHalf;
constexpr int kLdc = kTile + 16, kLdc32 = kTile + 4;
constexpr int kSideOff = kTile * kLdc * 2;  // the rows' and words' numbers for the epilogue, behind the tile
constexpr int kGemmSmem = kSideOff + kTile * 24;
static_assert(kSideOff >= 2 * kStage && kSideOff >= 128 * kLdc32 * 4, "the epilogues reuse the stages");
constexpr unsigned kOOB = 0x80000000u;     // past kRange: the load returns zeros
constexpr unsigned kRange = 0x7FFFFFF0u;

template <int N>
__device__ __forceinline__ void wait_vmcnt() {  // all but the wave's last N loads and stores are done
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// 16 bytes a lane from base + off (zeros past kRange) to the wave's 1 KiB at `dst` in LDS.  In assembly,
// because after the builtin the compiler waits for every fetch in flight before a transposed read of LDS;
// it has no register output, and wait_vmcnt is the wait for it.  base and dst are the wave's own.
__device__ __forceinline__ void fetch16(const u16* base, unsigned off, unsigned char* dst) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
  const u32x4 r = {static_cast<unsigned>(b), static_cast<unsigned>(b >> 32) & 0xFFFFu, kRange, 0x00020000u};
  const unsigned at = reinterpret_cast<uintptr_t>((lds_void*)dst);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 4\n\t"  // m0 needs one state, a scalar register that a vector instruction wrote five
      "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(r)
      : "memory", "m0");
}

// a barrier that leaves fetches in flight and that nothing is scheduled across
__device__ __forceinline__ void phase_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xC07F); }

__device__ __forceinline__ int xcd_remap(int bid, int nwg) {  // consecutive tiles on one XCD
  const int q = nwg >> 3, r = nwg & 7, x = bid & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (bid >> 3);
}
// Where 16-byte chunk ch of an image's row lies: at ch ^ swz(row), so that the fragment reads have no bank
// conflicts.  "Row" operands of two planes: 64-byte rows; of one: 128-byte rows; "col": [32 k][64 columns].
__device__ __forceinline__ int swz64_row(int row) { return (-(row >> 2)) & 3; }
__device__ __forceinline__ int swz128_row(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int swz128_col(int row) { return (((row >> 1) & 1) << 1) | (((row >> 3) & 1) << 2); }

// columns c0..c0+15 x 32 k of a [32][64] image: lane (g = lane >> 4, i = lane & 15) gets k 8g..8g+7 of column c0 + i
__device__ __forceinline__ s16x8 tr_frag(const unsigned char* sub, int c0, int lane) {
  const int g = lane >> 4, q = (lane >> 2) & 3, p = lane & 3;
  const int col = c0 + 4 * p;
  const int r0 = 8 * g + q, r1 = r0 + 4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sub + r0 * 128 + (((col >> 3) ^ swz128_col(r0)) << 4) + ((col & 4) << 1)));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sub + r1 * 128 + (((col >> 3) ^ swz128_col(r1)) << 4) + ((col & 4) << 1)));
  return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

template <bool F16>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// the value N lanes on in a row of 16
template <int N>
__device__ __forceinline__ float lane_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xF, 0xF, true));
}

// A wave's part of the tile, rounded to 16 bits, as rows of kLdc; two planes: what the rounding took 128 rows on.
// REST (one plane): what the rounding took, in place of the tile that is there.
template <bool F16, int PL, int FN, bool REST = false>
__device__ __forceinline__ void tile_to_lds(const f32x4 (&acc)[8][FN], unsigned char* smem, int row0, int col0) {
  typedef __attribute__((ext_vector_type(4))) u16 us4;
  u16* ct = reinterpret_cast<u16*>(smem);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      u16* o = ct + (row0 + i * 16) * kLdc + col0 + j * 16;
      us4 hi, lo;
      if (REST) lo = *reinterpret_cast<const us4*>(o);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = PL == 2 ? settled(acc[i][j][r]) : REST ? acc[i][j][r] - (F16 ? h2f(lo[r]) : bf2f(lo[r])) : acc[i][j][r];
        hi[r] = F16 ? f2h(v) : f2bf(v);
        if (PL == 2) lo[r] = f2h(v - h2f(hi[r]));
      }
      *reinterpret_cast<us4*>(o) = hi;
      if (PL == 2) *reinterpret_cast<us4*>(o + 128 * kLdc) = lo;
    }
}

// An exponential of at most 1 in 16 bits: five of exponent, down to 2^-31, and eleven behind the point, so it
// is off by at most 2^-12 of itself; zeros stand for what is smaller.
__device__ __forceinline__ u16 hold_bits(float e) {
  const int q = static_cast<int>((__float_as_uint(e) + 0x800u) >> 12) - (96 << 11);
  return static_cast<u16>(q < 0 ? 0 : q > 65535 ? 65535 : q);
}
__device__ __forceinline__ float held_value(unsigned q) { return q == 0 ? 0.f : __uint_as_float((q + (96u << 11)) << 12); }

// Where a block works: 256 rows from m0, 256 columns (or, of a tile cut in two, 128) from n0, k from kbeg to kend.
struct Place {
  int M, m0, n0, kbeg, kend, split;
  bool half, lone;  // 128 columns; and none beside them
};

// The blocks of a product: one a tile.  Fewer tiles than CUs: a sum (kPartial) is cut into pieces;
// otherwise, where the last round of 256 has at most half its CUs busy, its tiles are cut into two halves
// of 128 columns (a half takes about two thirds of a tile's time).  Counts depend on how many rows are
// kept, so a grid is sized for all of them and the blocks behind the last one return.
__device__ __forceinline__ int rows_of(const GemmArgs& g, int epi) {
  const int two = epi >= kPartial ? g.twice : 0;
  return g.m_dyn != nullptr ? *g.m_dyn << two : g.M;
}
__device__ __forceinline__ int sum_of(const GemmArgs& g) { return g.k_dyn != nullptr ? *g.k_dyn << g.twice : g.K; }

__device__ __forceinline__ int gemm_blocks(const GemmArgs& g, int epi) {
  const int M = rows_of(g, epi);
  const int tiles = ((M + kTile - 1) / kTile) * ((g.N + kTile - 1) / kTile);
  if (epi == kPartial && tiles < 256) {
    const int span = g.k_dyn != nullptr ? sum_of(g) : g.chunk;
    if (tiles == 0 || span == 0) return 0;
    const int len = split_length(tiles, span, g.least);
    return tiles * ((span + len - 1) / len);
  }
  const int last = tiles & 255;
  return tiles + (g.cut && last <= 128 ? last : 0);
}

__device__ __forceinline__ Place gemm_place(const GemmArgs& g, int epi, int bid, int blocks) {
  Place at;
  at.M = rows_of(g, epi);
  const int K = sum_of(g);
  const int ntm = (at.M + kTile - 1) / kTile, ntn = (g.N + kTile - 1) / kTile, tiles = ntm * ntn;
  at.split = at.kbeg = 0;
  at.kend = K;
  at.half = at.lone = false;
  int tile, side = 0;
  if (epi == kPartial && tiles < 256) {
    const int len = split_length(tiles, g.k_dyn != nullptr ? K : g.chunk, g.least);
    tile = xcd_remap(bid, blocks);
    at.split = tile / tiles;  // the tiles of one piece, which share its words, stay together
    tile -= at.split * tiles;
    at.kbeg = at.split * len;
    at.kend = at.kbeg + len < K ? at.kbeg + len : K;
  } else {
    const int whole = 2 * tiles - blocks;  // (blocks - tiles of them are cut)
    if (bid < whole) {
      tile = xcd_remap(bid, whole);
    } else {
      const int h = xcd_remap(bid - whole, blocks - whole);
      tile = whole + (h >> 1);
      side = h & 1;
      at.half = true;
    }
  }
  // tiles go down eight row tiles before they go on to the next column tile: what runs at one time
  // on an XCD then shares both operands
  const int per = 8 * ntn, band = tile / per, left = ntm - band * 8;
  const int high = left < 8 ? left : 8, in = tile - band * per;
  at.m0 = (band * 8 + in % high) * kTile;
  at.n0 = in / high * kTile;
  if (g.N - at.n0 <= 128) at.half = at.lone = true;
  at.n0 += side * 128;
  return at;
}

// One block's tile; FN: fragments of 16 columns a wave, 4, or 2 of a tile cut in two.
template <bool F16, int PL, bool ACOL, bool BCOL, int EPI, int FN>
__device__ __forceinline__ void gemm_tile(const GemmArgs& g, const Place& at, unsigned char* smem) {
  constexpr int KT = PL == 1 ? 64 : 32;  // k per stage
  constexpr int BN = FN * 64, JH = FN / 2;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid >> 2, wc = wid & 3;
  const int M = at.M, m0 = at.m0, n0 = at.n0, kbeg = at.kbeg, kend = at.kend;
  const int nk = kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0;

  // This lane's part of the four half tiles (0, 1: A; 2, 3: B): a wave fetches two 1 KiB pieces of each, q 0
  // of what a stage's first phase reads and q 1 of what only its second does (a "col" B: both for the first).
  // "Row" operands of one plane: 8 rows of 64 k, whole 128-byte lines; of two planes: 16 rows of 32 k of
  // either.  "Col" operands: 8 k rows of 64 columns.  Chunks are swizzled at the source.
  constexpr bool kBSplit = !BCOL && FN == 4;  // B's pieces in order of need: columns 0-31, then 32-63 of a wave
  unsigned voff[4][2];
  bool vok[4][2];
  int rk[4][2];  // k of a "row" piece's chunk, within the stage
  const int crow = (wid & 3) * 8 + (lane >> 3);
  auto piece_row = [&](int h, int q) {  // the first row of a "row" piece
    const int w = PL == 1 ? wid : wid >> 1, each = PL == 1 ? 8 : 16;
    if (h < 2 || !kBSplit) return q * 64 + w * each;
    return (w * each >> 5) * 64 + (w * each & 31) + q * 32;
  };
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const bool isa = h < 2, col = isa ? ACOL : BCOL;
      const int64_t ld = isa ? g.A.ld : g.B.ld;
      const int origin = isa ? m0 : n0, extent = isa ? M : g.N;
      if (!col) {
        const int row = piece_row(h, q) + (PL == 1 ? lane >> 3 : lane >> 2), r = (h & 1) * 128 + row;
        rk[h][q] = (PL == 1 ? (lane & 7) ^ swz128_row(row) : (lane & 3) ^ swz64_row(row)) * 8;
        vok[h][q] = origin + r < extent;
        voff[h][q] = static_cast<unsigned>(r * ld * 2 + rk[h][q] * 2);
      } else {
        const int c = (h & 1) * 128 + q * 64 + ((lane & 7) ^ swz128_col(crow)) * 8;
        rk[h][q] = 0;
        vok[h][q] = origin + c < extent;
        voff[h][q] = static_cast<unsigned>(crow * ld * 2 + c * 2);
      }
    }
  auto fetch = [&](int h, int q, int t) {
    const bool isa = h < 2, col = isa ? ACOL : BCOL;
    const Operand& op = isa ? g.A : g.B;
    const int part = col ? wid >> 2 : wid & 1;  // which 32 k, or which plane ("row" of one plane: neither)
    unsigned char* half = smem + (t & 1) * kStage + h * kHalf;
    const u16* base = op.p + (PL == 2 ? part * op.plane : 0);
    int k0 = kbeg + t * KT;
    bool ok;
    if (!col) {
      base += (isa ? m0 : n0) * op.ld + k0;
      ok = vok[h][q] && k0 + rk[h][q] < kend;
      half += PL == 1 ? piece_row(h, q) * 128 : part * 8192 + piece_row(h, q) * 64;
    } else {
      if (PL == 1) k0 += part * 32;
      base += k0 * op.ld + (isa ? m0 : n0);
      ok = vok[h][q] && k0 + crow < kend;
      half += part * 8192 + q * 4096 + (wid & 3) * 1024;
    }
    fetch16(base, ok ? voff[h][q] : kOOB, half);
  };
  // a stage's fetches in the order that they are issued in, two a group
  auto group = [&](int which, int t) {
    if (which == 0 || which == 3) {
      fetch(0, which & 1, t);
      fetch(1, which & 1, t);
    } else if (kBSplit) {
      fetch(2, which - 1, t);
      fetch(3, which - 1, t);
    } else if (FN == 4 || which == 1) {
      fetch(1 + which, 0, t);
      fetch(1 + which, 1, t);
    }
  };
  const int fr = lane & 15, fch = lane >> 4;
  // rows (or columns) r0 .. r0 + 15 of a half tile, part s: its k 32 s .. 32 s + 31, or its plane s
  auto frag = [&](bool col, const unsigned char* half, int r0, int s) -> s16x8 {
    if (col) return tr_frag(half + s * 8192 + (r0 >> 6) * 4096, r0 & 63, lane);
    const int r = r0 + fr;
    if (PL == 1) return *reinterpret_cast<const s16x8*>(half + r * 128 + (((s * 4 + fch) ^ swz128_row(r)) << 4));
    return *reinterpret_cast<const s16x8*>(half + s * 8192 + r * 64 + ((fch ^ swz64_row(r)) << 4));
  };

  // what the epilogue needs of each row (maximum, log of the sum, weight, target relative to the tile; scale) and
  // word (bias; -inf past the last) goes to LDS ahead of the products: there it would be loads in a row
  f32x4* side_row = reinterpret_cast<f32x4*>(smem + kSideOff);
  float* side_col = reinterpret_cast<float*>(smem + kSideOff + kTile * 16);
  int* side_e = reinterpret_cast<int*>(smem + kSideOff + kTile * 20);
  if constexpr (EPI == kStats || EPI == kGrad) {
    if (tid < kTile) {
      const int row = m0 + tid;
      f32x4 v = {0.f, 0.f, 0.f, __int_as_float(-1)};
      if (row < M) {
        if (EPI == kGrad) {
          v[0] = g.top[row];
          v[1] = g.log_s[row];
          v[2] = g.row_w != nullptr ? g.row_w[row] : g.g_scale;
        }
        if (g.words != nullptr) v[3] = __int_as_float(g.words[row] - g.v0 - n0);
      }
      if (PL == 2)
        side_e[tid] = row < M ? -scale_exp(static_cast<uint32_t>(g.bits[row])) - scale_exp(static_cast<uint32_t>(g.info[2])) : 0;
      side_row[tid] = v;
    } else if (tid < kTile + BN) {
      const int col = n0 + tid - kTile;
      side_col[tid - kTile] = col >= g.N ? kNegInf : g.bias != nullptr ? load_any(g.bias, col, g.bias_dt) : 0.f;
    }
  }

  f32x4 acc[8][FN];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Two stages (64 k, or 32 k of both planes), four phases a stage, a quadrant of the wave's tile each:
  // fragment reads and two fetches, a barrier, 16 or 24 matrix instructions (k halves 0 and 1; hi hi, hi lo,
  // lo hi), a barrier.  The lower four waves run one barrier late, so on every SIMD one wave multiplies while
  // the other reads and fetches.  All of a stage's fragments are in registers after its second phase.  A
  // place is fetched into again two phases after its last read: the stage after next's A for its first
  // phase in the third, B in the fourth and the next first, A for the second phase in the next second, so
  // that every phase issues as many (all eight in one phase held its barrier up); what a phase reads has
  // landed a phase before, with kAfterB or kAfterA fetches still on their way.
  constexpr int kAfterB = kBSplit ? 8 : 6, kAfterA = FN == 4 ? 6 : 4, kRest = kBSplit ? 4 : 2;
  s16x8 af[8][2], bf[FN][2];
  auto read_a = [&](int t, int i0) {
    const unsigned char* base = smem + (t & 1) * kStage + wr * kHalf;
#pragma unroll
    for (int i = i0; i < i0 + 4; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s) af[i][s] = frag(ACOL, base, i * 16, s);
  };
  auto read_b = [&](int t, int j0) {
    const int c0 = wc * (FN * 16);  // within the tile
    const unsigned char* base = smem + (t & 1) * kStage + (2 + (c0 >> 7)) * kHalf;
#pragma unroll
    for (int j = j0; j < j0 + JH; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) bf[j][s] = frag(BCOL, base, (c0 & 127) + j * 16, s);
  };
  auto mfma = [&](int i0, int j0) {
#pragma unroll
    for (int s = 0; s < (PL == 1 ? 2 : 3); ++s)
#pragma unroll
      for (int i = i0; i < i0 + 4; ++i)
#pragma unroll
        for (int j = j0; j < j0 + JH; ++j) acc[i][j] = mfma16<F16>(bf[j][PL == 1 ? s : s & 1], af[i][PL == 1 ? s : s >> 1], acc[i][j]);
  };
  if (nk > 0) {
    group(0, 0);
    group(1, 0);
    group(2, 0);
    group(3, 0);
    if (nk > 1) {
      group(0, 1);
      group(1, 1);
      wait_vmcnt<kAfterB>();
    } else {
      wait_vmcnt<kRest>();
    }
  }
  phase_barrier();
  if (wr == 1) phase_barrier();
  // Up to 128 rows left: 64-row quadrants behind the last one take no reads and no products (a row of 4096 against
  // 128000 words 235 to 173 us).  The conditions cost full tiles 2 to 7 % and a tile of 192 rows 2 %, so these have
  // a loop without.
  auto stages = [&](auto all) {
    const int left = M - m0 - wr * 128;
    const bool upper = all || left > 0, lower = all || left > 64;
    for (int t = 0; t < nk; ++t) {
      if (upper) {
        read_a(t, 0);
        read_b(t, 0);
      }
      if (t + 1 < nk) {
        group(2, t + 1);
        wait_vmcnt<kAfterA>();
      } else {
        wait_vmcnt<0>();
      }
      phase_barrier();
      wait_lgkm0();
      if (upper) mfma(0, 0);
      phase_barrier();
      if (lower) read_a(t, 4);
      if (upper) read_b(t, JH);
      if (t + 1 < nk) group(3, t + 1);
      phase_barrier();
      wait_lgkm0();
      if (upper) mfma(0, JH);
      phase_barrier();
      if (t + 2 < nk) group(0, t + 2);
      phase_barrier();
      if (lower) mfma(4, JH);
      phase_barrier();
      if (t + 2 < nk) {
        group(1, t + 2);
        wait_vmcnt<kAfterB>();
      } else {
        wait_vmcnt<kRest>();
      }
      phase_barrier();
      if (lower) mfma(4, 0);
      phase_barrier();
    }
  };
  if (M - m0 > 128) stages(std::true_type{});
  else stages(std::false_type{});
  if (wr == 0) phase_barrier();
  __syncthreads();

  // The tile is transposed in the accumulators (B is the instruction's first operand), so that a lane's
  // four consecutive values are of one row: acc[i][j][r] is row wr * 128 + i * 16 + fr, column
  // wc * 16 FN + j * 16 + fch * 4 + r.  A row's reduction is 4 FN values in registers and two lane steps.
  const int row0 = wr * 128 + fr, col0 = wc * (FN * 16) + fch * 4;
  if constexpr (EPI == kStats || EPI == kGrad) {
    auto logit = [&](float sum, float b, int unscale) { return (PL == 1 ? sum : times_pow2(sum, unscale)) + b; };
    const float c = g.c;
    f32x4 bias[4];
#pragma unroll
    for (int j = 0; j < FN; ++j) bias[j] = *reinterpret_cast<const f32x4*>(side_col + col0 + j * 16);
    if constexpr (EPI == kStats) {
      float* red = reinterpret_cast<float*>(smem);  // [3][4 column waves][256 rows]
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (m0 + wr * 128 + i * 16 >= M) break;  // nothing of the 16 rows' is read
        float m = kNegInf, s = 0.f, sz = 0.f;
        const int unscale = PL == 2 ? side_e[row0 + i * 16] : 0;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[i][j][r] = logit(acc[i][j][r], bias[j][r], unscale);
            m = fmaxf(m, acc[i][j][r]);
          }
        if (g.words != nullptr) {
          const int word = __float_as_int(side_row[row0 + i * 16][3]) - col0;  // j * 16 + r if the target is one of this lane's
          if (static_cast<unsigned>(word) < FN * 16u && (word & 15) < 4) {
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r) z = word == j * 16 + r ? acc[i][j][r] : z;
            g.picked[m0 + row0 + i * 16] = z;
          }
        }
        if (g.part_z != nullptr) {
#pragma unroll
          for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sz += n0 + col0 + j * 16 + r < g.N ? acc[i][j][r] * g.inv_v : 0.f;
          sz += __shfl_xor(sz, 16, 64);
          sz += __shfl_xor(sz, 32, 64);
        }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ref = m == kNegInf ? 0.f : m;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            acc[i][j][r] = exp2_((acc[i][j][r] - ref) * c);
            s += acc[i][j][r];
          }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (fch == 0) {
          const int to = wc * 256 + row0 + i * 16;
          red[to] = m;
          red[1024 + to] = s;
          red[2048 + to] = sz;
        }
      }
      __syncthreads();
      if (tid < 256 && m0 + tid < M) {
        float m = red[tid], s = red[1024 + tid], sz = red[2048 + tid];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          join(m, s, red[w * 256 + tid], red[1024 + w * 256 + tid], c);
          sz += red[2048 + w * 256 + tid];
        }
        // a place for every 128 columns; a whole tile fills two
        const int at128 = (g.v0 + n0) / 128;
        const int64_t to = static_cast<int64_t>(m0 + tid) * g.parts + at128;
        g.part[to] = make_float2(m, s);
        if (FN == 4 || at.lone) g.part[to + 1] = make_float2(kNegInf, 0.f);
        if (g.part_z != nullptr) {
          g.part_z[to] = sz;
          if (FN == 4 || at.lone) g.part_z[to + 1] = 0.f;
        }
        if (g.E != nullptr && g.v0 + n0 < g.held) {
          float* tops = g.tops + static_cast<int64_t>(m0 + tid) * (g.held / 128) + at128;
          tops[0] = m;
          if (FN == 4 || at.lone) tops[1] = m;
        }
      }
      if (g.E != nullptr && g.v0 + n0 < g.held) {
        // e = 2^(c (z - the tile's maximum)), from those below the wave's
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float own = red[wc * 256 + row0 + i * 16];
          const float m = fmaxf(fmaxf(red[row0 + i * 16], red[256 + row0 + i * 16]), fmaxf(red[512 + row0 + i * 16], red[768 + row0 + i * 16]));
          const float f = own == kNegInf ? 0.f : exp2_((own - m) * c);
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] *= f;
        }
        __syncthreads();
        if (PL == 1 && !g.exact) {
          typedef __attribute__((ext_vector_type(4))) u16 us4;
          u16* ct = reinterpret_cast<u16*>(smem);
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
              us4 v;
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] = hold_bits(acc[i][j][r]);
              *reinterpret_cast<us4*>(ct + (row0 + i * 16) * kLdc + col0 + j * 16) = v;
            }
          __syncthreads();
          u16* out = static_cast<u16*>(g.E) + g.v0 + n0;
          for (int q = tid; q < kTile * (BN / 8); q += kThreads) {
            const int row = q / (BN / 8), cc = (q % (BN / 8)) * 8;
            if (m0 + row < M)
              *reinterpret_cast<us8*>(out + static_cast<int64_t>(m0 + row) * g.held + cc) =
                  *reinterpret_cast<const us8*>(ct + row * kLdc + cc);
          }
        } else {
          float* ct = reinterpret_cast<float*>(smem);  // half the rows at a time
          float* out = static_cast<float*>(g.E) + g.v0 + n0;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (wr == half)
#pragma unroll
              for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) *reinterpret_cast<f32x4*>(ct + (fr + i * 16) * kLdc32 + col0 + j * 16) = acc[i][j];
            __syncthreads();
            for (int q = tid; q < 128 * (BN / 4); q += kThreads) {
              const int row = half * 128 + q / (BN / 4), cc = (q % (BN / 4)) * 4;
              if (m0 + row < M)
                *reinterpret_cast<f32x4*>(out + static_cast<int64_t>(m0 + row) * g.held + cc) =
                    *reinterpret_cast<const f32x4*>(ct + (row - half * 128) * kLdc32 + cc);
            }
            __syncthreads();
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool ok = m0 + row0 + i * 16 < M;
        const f32x4 of = side_row[row0 + i * 16];
        const float top = of[0], l = of[1], w = of[2];
        const int unscale = PL == 2 ? side_e[row0 + i * 16] : 0;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = exp2_(fmaf(logit(acc[i][j][r], bias[j][r], unscale) - top, c, -l));
            acc[i][j][r] = ok ? w * (p - g.smooth_v) : 0.f;
          }
        if (g.words != nullptr) {
          const int word = __float_as_int(of[3]) - col0;
          if (static_cast<unsigned>(word) < FN * 16u && (word & 15) < 4) {
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][r] -= word == j * 16 + r ? w * g.share : 0.f;
          }
        }
      }
      if (g.colsum != nullptr) {  // before G is rounded
        float* red = reinterpret_cast<float*>(smem);  // [2 row waves][256 columns]
        float each[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = m0 + row0 + i * 16;
          each[i] = g.row_e != nullptr && row < M ? times_pow2(1.f, g.row_e[row]) : 1.f;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          f32x4 t = acc[0][j] * each[0];
#pragma unroll
          for (int i = 1; i < 8; ++i) t += acc[i][j] * each[i];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            t[r] += lane_ror<8>(t[r]);
            t[r] += lane_ror<4>(t[r]);
            t[r] += lane_ror<2>(t[r]);
            t[r] += lane_ror<1>(t[r]);
          }
          if (fr == 0) *reinterpret_cast<f32x4*>(red + wr * 256 + col0 + j * 16) = t;
        }
        __syncthreads();
        if (tid < BN && n0 + tid < g.ldg) g.colsum[static_cast<int64_t>(m0 / kTile) * g.ldg + n0 + tid] = red[tid] + red[256 + tid];
        __syncthreads();
      }
      // one plane: the whole tile through LDS, and again if G's rows are two; two: both planes of half the
      // rows at a time
      const int rows = kTile / PL;
      auto pass = [&](int half) {
        const int to = PL == 1 ? half * M : half * rows;
        __syncthreads();
        for (int q = tid; q < kTile * (BN / 8); q += kThreads) {
          const int line = q / (BN / 8), cc = (q % (BN / 8)) * 8, pl = line / rows, row = m0 + line % rows;
          if (row + (PL == 1 ? 0 : to) < M && n0 + cc < g.ldg)
            *reinterpret_cast<us8*>(g.G + pl * g.g_plane + static_cast<int64_t>(row + to) * g.ldg + n0 + cc) =
                *reinterpret_cast<const us8*>(reinterpret_cast<const u16*>(smem) + line * kLdc + cc);
        }
      };
      if (PL == 1 || wr == 0) tile_to_lds<F16, PL>(acc, smem, PL == 1 ? row0 : fr, col0);
      pass(0);
      if (PL == 2 || g.twice) {
        __syncthreads();
        if (PL == 1) tile_to_lds<F16, 1, FN, true>(acc, smem, row0, col0);
        else if (wr == 1) tile_to_lds<F16, PL>(acc, smem, fr, col0);
        pass(1);
      }
    }
  } else if constexpr (EPI == kPartial) {
    float* out = g.out32 + at.split * (M * g.ldo);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int row = m0 + row0 + i * 16;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int col = n0 + col0 + j * 16;
        if (row < M && col < g.ldo) {
          f32x4* o = reinterpret_cast<f32x4*>(out + row * g.ldo + col);
          f32x4 v = acc[i][j];
          if (g.add) v += *o;
          *o = v;
        }
      }
    }
  } else {
    const float alpha = g.alpha();
    const int unscale = PL == 1 ? 0 : -scale_exp(static_cast<uint32_t>(*g.bits));
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = PL == 1 ? acc[i][j][r] * alpha : times_pow2(acc[i][j][r] * alpha, unscale);
    if constexpr (PL == 1) {
      tile_to_lds<F16, 1>(acc, smem, row0, col0);
      __syncthreads();
      const u16* ct = reinterpret_cast<const u16*>(smem);
      u16* out = static_cast<u16*>(g.out);
      // 16-byte stores need no alignment here, so rows of any width take them
      for (int q = tid; q < kTile * (BN / 8); q += kThreads) {
        const int row = q / (BN / 8), cc = (q % (BN / 8)) * 8, left = g.N - n0 - cc;
        if (m0 + row >= M) continue;
        u16* o = out + (m0 + row) * g.ldo + n0 + cc;
        if (left >= 8) __builtin_memcpy(o, ct + row * kLdc + cc, 16);
        else
          for (int e = 0; e < left; ++e) o[e] = ct[row * kLdc + cc + e];
      }
    } else {
      float* ct = reinterpret_cast<float*>(smem);  // half the rows at a time
      float* out = static_cast<float*>(g.out);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (wr == half)
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) *reinterpret_cast<f32x4*>(ct + (fr + i * 16) * kLdc32 + col0 + j * 16) = acc[i][j];
        __syncthreads();
        for (int q = tid; q < 128 * (BN / 4); q += kThreads) {
          const int row = q / (BN / 4), cc = (q % (BN / 4)) * 4, left = g.N - n0 - cc;
          if (m0 + half * 128 + row >= M) continue;
          float* o = out + (m0 + half * 128 + row) * g.ldo + n0 + cc;
          if (left >= 4) __builtin_memcpy(o, ct + row * kLdc32 + cc, 16);
          else
            for (int e = 0; e < left; ++e) o[e] = ct[row * kLdc32 + cc + e];
        }
        __syncthreads();
      }
    }
  }
}

template <bool F16, int PL, bool ACOL, bool BCOL, int EPI>
__device__ __forceinline__ void gemm_block(const GemmArgs& g, int bid, int blocks, unsigned char* smem) {
  const Place at = gemm_place(g, EPI, bid, blocks);
  if (at.n0 >= g.N) return;  // the other half of a lone one
  if (at.half) gemm_tile<F16, PL, ACOL, BCOL, EPI, 2>(g, at, smem);
  else gemm_tile<F16, PL, ACOL, BCOL, EPI, 4>(g, at, smem);
}

template <bool F16, int PL, bool ACOL, bool BCOL, int EPI>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(GemmArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int blocks = gemm_blocks(g, EPI);
  if (static_cast<int>(blockIdx.x) < blocks) gemm_block<F16, PL, ACOL, BCOL, EPI>(g, blockIdx.x, blocks, smem);
#endif
}


// The statistics of few tiles of logits, whose sums over D came in pieces (kPartial, of g.chunk): what kStats'
// epilogue does, a wave for 256 words of a row.  Bound by reading the pieces (482 x 2738, ten of them: 53 MB from
// the caches in 11 us).
__global__ void __launch_bounds__(256) pieces_kernel(GemmArgs g, int planes) {
  const int M = *g.m_dyn, ntn = (g.N + kTile - 1) / kTile, lane = threadIdx.x & 63;
  if (M == 0) return;
  const int len = split_length((M + kTile - 1) / kTile * ntn, g.chunk, g.least), splits = (g.chunk + len - 1) / len;
  const int of_words = planes == 1 ? 0 : -scale_exp(static_cast<uint32_t>(g.info[2]));
  const int64_t units = static_cast<int64_t>(M) * ntn, stride = M * g.ldo;
  for (int64_t unit = blockIdx.x * 4ll + (threadIdx.x >> 6); unit < units; unit += gridDim.x * 4ll) {
    const int row = static_cast<int>(unit / ntn), tile = static_cast<int>(unit - static_cast<int64_t>(row) * ntn);
    const int col = tile * kTile + lane * 4;
    const int unscale = planes == 1 ? 0 : of_words - scale_exp(static_cast<uint32_t>(g.bits[row]));
    const float* p = g.out32 + row * g.ldo + col;
    f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) z += *reinterpret_cast<const f32x4*>(p + s * stride);
    float m = kNegInf, sum = 0.f, sz = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool there = col + e < g.N;
      z[e] = there ? times_pow2(z[e], unscale) + (g.bias != nullptr ? load_any(g.bias, col + e, g.bias_dt) : 0.f) : kNegInf;
      if (there) sz += z[e] * g.inv_v;
      m = fmaxf(m, z[e]);
    }
    m = max_lanes(m);
    const float ref = m == kNegInf ? 0.f : m;
    const int word = g.words != nullptr ? g.words[row] - col : -1;
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (word == e) g.picked[row] = z[e];
      x[e] = exp2_((z[e] - ref) * g.c);
      sum += x[e];
    }
    sum = sum_lanes(sum);
    if (g.part_z != nullptr) sz = sum_lanes(sz);
    if (lane < 2) {
      const int64_t to = static_cast<int64_t>(row) * g.parts + tile * 2 + lane;
      g.part[to] = lane == 0 ? make_float2(m, sum) : make_float2(kNegInf, 0.f);
      if (g.part_z != nullptr) g.part_z[to] = lane == 0 ? sz : 0.f;
      if (g.E != nullptr) g.tops[static_cast<int64_t>(row) * (g.held / 128) + tile * 2 + lane] = m;
    }
    if (g.E == nullptr) continue;
    const int64_t at = static_cast<int64_t>(row) * g.held + col;
    if (g.exact) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(g.E) + at) = x;
    } else {
      typedef __attribute__((ext_vector_type(4))) u16 us4;
      us4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = hold_bits(x[e]);
      *reinterpret_cast<us4*>(static_cast<u16*>(g.E) + at) = v;
    }
  }
}

// ------------------------------------------------------------------------------------------------
// Joining a row's tiles, its K picked logits, its loss.  One wave a row (cross entropy) or four (lists).
// ------------------------------------------------------------------------------------------------
struct FinishArgs {
  const void *x, *w, *bias;
  int64_t x_ld, w_ld;
  int dt, bias_dt, D, V, K, parts, N;
  const int *info, *list;
  const float2* part;
  const float* part_z;
  const int* words;    // one target a row
  const void *index, *teacher;
  int64_t index_ld, teacher_ld;
  int wide, teacher_dt;
  float inv_t, smooth;
  float *top, *log_s;  // [kept]
  float* picked;       // [kept][K] logits of the picked words (a target's: from the product)
  float* share;        // [kept][K]
  double* rows;        // losses [kept], for a mean or a sum (a row's may be past fp32 where their mean is not)
  float* each;         // losses [N], or null
};

// x . w for four weight rows at a time, by one wave; nothing stands between the loads of a step
template <int DT>
__device__ __forceinline__ void dots_wave(const typename Elem<DT>::type* x, const typename Elem<DT>::type* const (&w)[4], int D, int lane,
                                          float (&out)[4]) {
  typedef typename Elem<DT>::type T;
#pragma unroll
  for (int q = 0; q < 4; ++q) out[q] = 0.f;
  auto step = [&](int d, int there) {
    T a[8], b[4][8];
    load8(x + d, there, a);
#pragma unroll
    for (int q = 0; q < 4; ++q) load8(w[q] + d, there, b[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 8; ++e) out[q] = fmaf(to_f<DT>(a[e]), to_f<DT>(b[q][e]), out[q]);
  };
  const int whole = D & ~511;
#pragma unroll 2
  for (int d = 0; d < whole; d += 512) step(d + lane * 8, 8);
  if (whole + lane * 8 < D) step(whole + lane * 8, D - whole - lane * 8);
#pragma unroll
  for (int q = 0; q < 4; ++q) out[q] = sum_lanes(out[q]);
}

// an entry of a teacher's list: absent if its word is negative or its logit -inf
__device__ __forceinline__ bool list_entry(const void* index, int64_t at, int wide, const void* teacher, int64_t t_at, int t_dt,
                                           int64_t& word, float& t) {
  word = load_index(index, at, wide);
  t = load_any(teacher, t_at, t_dt);
  return word >= 0 && t != kNegInf;
}
// one entry's part of the divergence / T^2: q (log q - log p), q = 2^(c (t - tt) - tl), log p = (z - top) / T - ln 2 log_s
__device__ __forceinline__ float diverge(float q, float t, float tt, float tl, float z, float top, float log_s, float inv_t) {
  if (q == 0.f) return 0.f;
  return q * (((t - tt) * inv_t - tl * kLn2) - ((z - top) * inv_t - log_s * kLn2));
}

// one target a row: a wave each (8192 rows of 1000 parts in 18 us, one row in 5)
__global__ void __launch_bounds__(256) finish_target_kernel(FinishArgs a) {
  const int lane = threadIdx.x & 63, count = a.info[0];
  for (int row = blockIdx.x * 4 + (threadIdx.x >> 6); row < count; row += gridDim.x * 4) {
    float m = kNegInf, s = 0.f, sz = 0.f;
    const int64_t at = static_cast<int64_t>(row) * a.parts;
    for (int t = lane; t < a.parts; t += 512) {  // eight loads on their way at a time
      float2 v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = t + e * 64 < a.parts ? a.part[at + t + e * 64] : make_float2(kNegInf, 0.f);
#pragma unroll
      for (int e = 0; e < 8; ++e) join(m, s, v[e].x, v[e].y, kLog2e);
      if (a.part_z != nullptr)
#pragma unroll
        for (int e = 0; e < 8; ++e) sz += t + e * 64 < a.parts ? a.part_z[at + t + e * 64] : 0.f;
    }
    join_lanes(m, s, 64, kLog2e);
    if (a.part_z != nullptr) sz = sum_lanes(sz);
    if (lane == 0) {
      const float log_s = log2f(s);
      // a word outside the vocabulary: the row's loss and gradients are NaN
      const float z = a.words[row] >= 0 ? a.picked[row] : __builtin_nanf("");
      // with eps = 1 the target does not count, not even one of logit -inf
      float loss = log_s * kLn2;
      if (a.smooth != 1.f || z != z) loss += (1.f - a.smooth) * (m - z);
      if (a.smooth != 0.f) loss += a.smooth * (m - sz);
      a.top[row] = m;
      a.log_s[row] = loss != loss ? loss : log_s;
      if (a.each != nullptr) a.each[a.list[row]] = loss;
      else a.rows[row] = loss;
    }
  }
}

// a list a row: a block each, four waves with four words' rows at a time (2048 x 64 words of 2048 bf16, 537 MB
// from the caches, in 76 us)
template <int DT>
__global__ void __launch_bounds__(256) finish_list_kernel(FinishArgs a) {
  __shared__ float red[4][3];
  typedef typename Elem<DT>::type T;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int count = a.info[0];
  const float c = a.inv_t * kLog2e;
  for (int row = blockIdx.x; row < count; row += gridDim.x) {
    const int n = a.list[row];
    float m = kNegInf, s = 0.f;
    for (int t = tid; t < a.parts; t += 256) {
      const float2 v = a.part[static_cast<int64_t>(row) * a.parts + t];
      join(m, s, v.x, v.y, c);
    }
    join_lanes(m, s, 64, c);
    __syncthreads();
    if (lane == 0) {
      red[wv][0] = m;
      red[wv][1] = s;
    }
    __syncthreads();
    m = red[0][0];
    s = red[0][1];
    for (int w = 1; w < 4; ++w) join(m, s, red[w][0], red[w][1], c);
    const float log_s = log2f(s);
    const T* x = static_cast<const T*>(a.x) + n * a.x_ld;
    const int64_t i0 = n * a.index_ld, t0 = n * a.teacher_ld, k0 = static_cast<int64_t>(row) * a.K;
    float tt = kNegInf, ts = 0.f;
    for (int k = lane; k < a.K; k += 64) {  // every wave goes over the whole list
      int64_t word;
      float t;
      if (list_entry(a.index, i0 + k, a.wide, a.teacher, t0 + k, a.teacher_dt, word, t)) join(tt, ts, t, 1.f, c);
    }
    join_lanes(tt, ts, 64, c);
    const float tl = log2f(ts);
    float loss = 0.f;  // this wave's part
    for (int k = wv * 4; k < a.K; k += 16) {
      const T* w[4];
      int64_t word[4];
      float t[4], z[4];
      bool there[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        there[q] = k + q < a.K && list_entry(a.index, i0 + k + q, a.wide, a.teacher, t0 + k + q, a.teacher_dt, word[q], t[q]);
        w[q] = static_cast<const T*>(a.w) + (there[q] && word[q] < a.V ? word[q] : 0) * a.w_ld;  // (absent: any row, not used)
      }
      dots_wave<DT>(x, w, a.D, lane, z);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float share = 0.f;
        if (there[q]) {
          share = exp2_(fmaf(t[q] - tt, c, -tl));
          // a word outside the vocabulary: the row's loss and gradients are NaN
          if (word[q] >= a.V) {
            loss = __builtin_nanf("");
            z[q] = 0.f;
          } else if (a.bias != nullptr) {
            z[q] += load_any(a.bias, word[q], a.bias_dt);
          }
          loss += diverge(share, t[q], tt, tl, z[q], m, log_s, a.inv_t);
        }
        if (lane == 0 && k + q < a.K) {
          a.picked[k0 + k + q] = z[q];
          a.share[k0 + k + q] = share;
        }
      }
    }
    if (lane == 0) red[wv][2] = loss;
    __syncthreads();
    if (tid == 0) {
      const float t = (red[0][2] + red[1][2]) + (red[2][2] + red[3][2]);
      a.top[row] = m;
      a.log_s[row] = t != t ? t : log_s;
      const double all = static_cast<double>(t) / (static_cast<double>(a.inv_t) * a.inv_t);
      if (a.each != nullptr) a.each[n] = static_cast<float>(all);
      else a.rows[row] = all;
    }
  }
}

// sum of the kept rows' losses, or their mean (nothing kept: 0)
__global__ void __launch_bounds__(1024) reduce_kernel(const double* rows, const int* info, int mean, float* out) {
  __shared__ double part[16];
  const int count = info[0];
  double s = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) s += rows[i];
  for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += part[w];
    *out = static_cast<float>(mean && count > 0 ? s / count : s);
  }
}

// ------------------------------------------------------------------------------------------------
// Backward of losses by row: row_w[c] 2^row_e[c] = g_n / max |g| times 2^kGExp for fp16 G, *top = max |g|, over the
// rows whose g is finite: one that is not keeps its own, and spoils no other row.  (A mean and a sum have one weight for
// all, and need none of this.)
// G in fp16 has its smallest step at 2^-38.  A row whose weight is below 2^-8 of the largest would lose its bits
// there, so its row_w is taken back to 2^-8..2^-7 and row_e says how far: G w is multiplied by it at the end, and for
// G^T h it goes into h, whose rows are packed once more (to 2^-25 of the largest weight for fp16, 2^-39 of the
// largest h for fp32: what a row of a far smaller weight gives to a sum over rows).  bf16 has fp32's range and needs none.
// ------------------------------------------------------------------------------------------------
struct WeightArgs {
  const float* g;  // [N]
  const int *info, *list;
  float *row_w, *top;
  int* row_e;      // null: zeros
  const int* each; // fp32: the largest magnitude of each row of h; *most: of them times 2^row_e
  int* most;
  float g_scale;
};

__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u; }

__global__ void __launch_bounds__(1024) weights_kernel(WeightArgs a) {
  __shared__ float part[16];
  const int count = a.info[0];
  float top = 0.f, most = 0.f;
  for (int c = threadIdx.x; c < count; c += 1024) {
    const float g = fabsf(a.g[a.list[c]]);
    if (finite(g)) top = fmaxf(top, g);
  }
  top = max_lanes(top);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  top = part[0];
  for (int w = 1; w < 16; ++w) top = fmaxf(top, part[w]);
  for (int c = threadIdx.x; c < count; c += 1024) {
    const float g = a.g[a.list[c]];
    int e = 0;
    if (a.row_e != nullptr) {
      if (finite(g) && g != 0.f) e = __builtin_amdgcn_frexp_expf(g) - __builtin_amdgcn_frexp_expf(top) + 8;
      a.row_e[c] = e = e < 0 ? e : 0;
    }
    a.row_w[c] = !finite(g) ? g : top == 0.f ? 0.f : times_pow2(g, -e) / top * a.g_scale;
    if (a.each != nullptr) most = fmaxf(most, times_pow2(__int_as_float(a.each[c]), e));
  }
  if (threadIdx.x == 0) *a.top = top;
  if (a.each == nullptr) return;
  most = max_lanes(most);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) most = fmaxf(most, part[w]);
    *a.most = __float_as_int(most);
  }
}

// ------------------------------------------------------------------------------------------------
// G of the words whose exponentials the forward pass left: w (e 2^(c (the tile's maximum - top) - log2 sum) -
// eps / V), minus the target's share; as the product's epilogue writes it.  A block has 256 rows of 64
// words, eight lanes a row.  Bound by memory (2048 x 32000, 2 bytes in and 2 out: 54 us, 4.9 TB/s).
// ------------------------------------------------------------------------------------------------
struct HeldArgs {
  const void* E;
  const float* tops;
  int held;       // (a multiple of 256)
  const int* info;
  const float *top, *log_s, *row_w;
  const int* row_e;
  float g_scale, c, smooth_v, share;
  const int* words;  // one target a row (null for lists)
  int v0;
  float* colsum;     // [tiles of rows][ldg] or null
  u16* G;
  int64_t g_plane;
  int ldg, twice;
};

template <int DT, bool EXACT>
__global__ void __launch_bounds__(256) held_kernel(HeldArgs a) {
  constexpr bool kF = DT == kF32;
  const int M = a.info[0], tid = threadIdx.x, across = a.ldg / 64, down = static_cast<int>(blockIdx.x) / across;
  const int col0 = (static_cast<int>(blockIdx.x) - down * across) * 64, col = col0 + (tid & 7) * 8, m0 = down * kTile;
  if (m0 >= M) return;
  float sums[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int it = 0; it < 8; ++it) {
    const int row = m0 + it * 32 + (tid >> 3);
    if (row >= M) continue;
    const int64_t at = static_cast<int64_t>(row) * a.held + col;
    float g[8];
    if constexpr (EXACT) {
      const f32x4* e = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.E) + at);
      const f32x4 lo = __builtin_nontemporal_load(e), hi = __builtin_nontemporal_load(e + 1);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        g[k] = lo[k];
        g[k + 4] = hi[k];
      }
    } else {
      const us8 e = __builtin_nontemporal_load(reinterpret_cast<const us8*>(static_cast<const u16*>(a.E) + at));
#pragma unroll
      for (int k = 0; k < 8; ++k) g[k] = held_value(e[k]);
    }
    const float w = a.row_w != nullptr ? a.row_w[row] : a.g_scale;
    const float tile = a.tops[static_cast<int64_t>(row) * (a.held / 128) + col / 128];
    const float f = exp2_(fmaf(tile - a.top[row], a.c, -a.log_s[row]));
    const int word = a.words != nullptr ? a.words[row] - a.v0 - col : -1;
    const float each = a.row_e != nullptr ? times_pow2(1.f, a.row_e[row]) : 1.f;
    us8 hi, lo;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      g[k] = settled(w * (fmaf(g[k], f, -a.smooth_v) - (word == k ? a.share : 0.f)));
      sums[k] += g[k] * each;
      hi[k] = DT == kBF16 ? f2bf(g[k]) : f2h(g[k]);
      lo[k] = DT == kBF16 ? f2bf(g[k] - bf2f(hi[k])) : f2h(g[k] - h2f(hi[k]));
    }
    u16* o = a.G + static_cast<int64_t>(row) * a.ldg + col;
    *reinterpret_cast<us8*>(o) = hi;
    if (kF) *reinterpret_cast<us8*>(o + a.g_plane) = lo;
    else if (a.twice) *reinterpret_cast<us8*>(o + static_cast<int64_t>(M) * a.ldg) = lo;
  }
  if (a.colsum == nullptr) return;
  __shared__ float red[32][64 + 4];
#pragma unroll
  for (int k = 0; k < 8; ++k) red[tid >> 3][(tid & 7) * 8 + k] = sums[k];
  __syncthreads();
  if (tid < 64) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += red[r][tid];
    a.colsum[static_cast<int64_t>(down) * a.ldg + col0 + tid] = t;
  }
}

// The listed words' entries of a chunk's G, from the fp32 logits of the forward pass (a word twice in a list: its
// shares add up, and each of its entries writes the same value), and their part of the bias gradient.  Each entry goes
// over its row's list for that, so the work grows with K^2: 2048 lists of 64 in 16 us, a step of them with K = 1024
// takes 3.2 ms where K = 64 takes 0.95.
struct ScatterArgs {
  const int *info, *list;
  const void* index;
  int64_t index_ld;
  int wide, K, v0, nv, f16, planes, ldg;
  const float *picked, *share, *top, *log_s, *row_w;
  const int* row_e;
  float g_scale, c;
  u16* G;
  int64_t g_plane;
  int twice;
  unsigned long long* listed;  // [nv] sums of shares times their rows' weights, in whole steps, or null
  double steps;                // steps of a weight g_scale
};

__global__ void __launch_bounds__(256) clear_kernel(unsigned long long* p, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

__global__ void __launch_bounds__(256) scatter_kernel(ScatterArgs a) {
  const int count = a.info[0];
  const int64_t all = static_cast<int64_t>(count) * a.K;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < all; i += gridDim.x * 256ll) {
    const int row = static_cast<int>(i / a.K), k = static_cast<int>(i - static_cast<int64_t>(row) * a.K);
    const int64_t i0 = a.list[row] * a.index_ld, word = load_index(a.index, i0 + k, a.wide);
    const float* share = a.share + static_cast<int64_t>(row) * a.K;
    if (word < a.v0 || word >= a.v0 + a.nv || share[k] == 0.f) continue;  // no share: another entry's, or p alone
    float s = 0.f;
    for (int j = 0; j < a.K; ++j)
      if (load_index(a.index, i0 + j, a.wide) == word) s += share[j];
    const float w = a.row_w != nullptr ? a.row_w[row] : a.g_scale;
    // integers, whose sum does not depend on their order (a row that is not finite shows in p's part)
    if (a.listed != nullptr && finite(w * share[k]))
      atomicAdd(a.listed + (word - a.v0), static_cast<unsigned long long>(__double2ll_rn(
                                              __builtin_ldexp(static_cast<double>(w) * share[k] * a.steps, a.row_e != nullptr ? a.row_e[row] : 0))));
    const float v = settled(w * (exp2_(fmaf(a.picked[i] - a.top[row], a.c, -a.log_s[row])) - s));
    u16* o = a.G + static_cast<int64_t>(row) * a.ldg + (word - a.v0);
    const u16 hi = a.f16 ? f2h(v) : f2bf(v);
    *o = hi;
    if (a.planes == 2) o[a.g_plane] = f2h(v - h2f(hi));
    else if (a.twice) o[static_cast<int64_t>(count) * a.ldg] = a.f16 ? f2h(v - h2f(hi)) : f2bf(v - bf2f(hi));
  }
}

// the bias gradient: column sums of G before its rounding, one for every tile of kept rows, less the shares of listed words
__global__ void __launch_bounds__(256) dbias_kernel(const float* part, int ldg, int nv, const unsigned long long* listed, double steps,
                                                    Alpha alpha, void* db, int64_t at, int dt) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= nv) return;
  const int splits = (alpha.info[0] + kTile - 1) / kTile;
  float t = 0.f;
#pragma unroll 8
  for (int s = 0; s < splits; ++s) t += part[static_cast<int64_t>(s) * ldg + v];
  if (listed != nullptr) t = static_cast<float>(t - static_cast<double>(static_cast<long long>(listed[v])) / steps);
  store_any(db, at + v, dt, t * alpha());
}

// The sum of a row's partials: of dh (pos: a row's place among the kept ones; zeros for the others), or of
// dw (pos null; rows of words, pieces of the kept rows).  Bound by memory (4608 rows, 28 pieces of 691 kept:
// 59 MB in 13 us)
__global__ void __launch_bounds__(256) sum_kernel(const float* part, int span, int64_t ldo, const int* info, const int* bits, const int* pos,
                                                  const int* row_e, int twice, Alpha alpha, int planes, void* dx, int dt, int D) {
  const int n = blockIdx.x, at = pos != nullptr ? pos[n] : n, count = pos != nullptr ? info[0] << twice : gridDim.x;
  const int tiles = ((count + kTile - 1) / kTile) * ((D + kTile - 1) / kTile);
  int splits = 0;
  if (pos == nullptr) span = info[0];
  if (at >= 0 && span > 0) {
    const int len = split_length(tiles, span, kPiece);
    splits = (span + len - 1) / len;
  }
  const float a = at >= 0 ? alpha() : 0.f;  // (a row that does not count: zeros, whatever the derivative is)
  int unscale = planes == 2 ? -scale_exp(static_cast<uint32_t>(*bits)) : 0;
  if (row_e != nullptr && at >= 0) unscale += row_e[at];
  const int64_t stride = count * ldo, out = static_cast<int64_t>(n) * D;
  for (int d = (blockIdx.y * 256 + threadIdx.x) * 4; d < D; d += gridDim.y * 1024) {
    f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* p = part + at * ldo + d;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) t += *reinterpret_cast<const f32x4*>(p + s * stride);
    if (twice)
#pragma unroll 4
      for (int s = 0; s < splits; ++s) t += *reinterpret_cast<const f32x4*>(p + info[0] * ldo + s * stride);
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = times_pow2(t[e] * a, unscale);
    if (d + 4 <= D) {  // (wide stores need no alignment)
      if (dt == kF32) {
        __builtin_memcpy(static_cast<float*>(dx) + out + d, &t, 16);
      } else {
        typedef __attribute__((ext_vector_type(4))) u16 us4;
        us4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = dt == kBF16 ? f2bf(t[e]) : f2h(t[e]);
        __builtin_memcpy(static_cast<u16*>(dx) + out + d, &o, 8);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < D) store_any(dx, out + d + e, dt, t[e]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// A teacher's top logits against logits in memory: reads them once forward, once backward.
// ------------------------------------------------------------------------------------------------
struct LogitArgs {
  const void* z;
  int64_t z_ld;
  int dt, N, V, K, segs, seg_len;  // seg_len % 8 == 0
  const void *index, *teacher;
  int64_t index_ld, teacher_ld;
  int wide, teacher_dt;
  float inv_t;
  int each, mean;
  float2* part;        // [N][segs]
  float *top, *log_s;  // [N]; a log_s of +inf marks a row without a list (every p 0)
  float* share;        // [N][K]
  double* rows;        // [N]
  float* loss_each;    // [N], or null
  int* info;     // [0]: rows with a list
  // backward
  const float* g;
  void* dz;
  int64_t dz_ld;
  int stream;  // whether dz is more than the caches hold
};

// One pass over a segment, four 16-byte pieces a thread in flight: f(column, its W values) for the whole
// pieces from the first 16-byte boundary on, f1(column, value) for what is before and behind them.
template <int DT, class F, class F1>
__device__ __forceinline__ void walk(const typename Elem<DT>::type* p, int lo, int hi, int tid, F&& f, F1&& f1) {
  typedef typename Elem<DT>::type T;
  constexpr int W = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(W))) T V;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(p + lo) & 15) / sizeof(T));
  int start = lo + (mis ? W - mis : 0);
  if (start > hi) start = hi;
  const int whole = (hi - start) / W, rest = start + whole * W;
  if (tid < start - lo) f1(lo + tid, p[lo + tid]);
  if (tid < hi - rest) f1(rest + tid, p[rest + tid]);
  const V* q = reinterpret_cast<const V*>(p + start);
  int i = tid;
  for (; i + 3 * 256 < whole; i += 4 * 256) {
    V v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = q[i + u * 256];
#pragma unroll
    for (int u = 0; u < 4; ++u) f(start + (i + u * 256) * W, v[u]);
  }
  for (; i < whole; i += 256) f(start + i * W, q[i]);
}

// whether a row's list has an entry (every wave of a block finds the same)
__device__ __forceinline__ bool has_list(const LogitArgs& a, int n, int lane) {
  bool any = false;
  for (int k = lane; k < a.K; k += 64) {
    int64_t word;
    float t;
    any |= list_entry(a.index, n * a.index_ld + k, a.wide, a.teacher, n * a.teacher_ld + k, a.teacher_dt, word, t);
  }
  return __ballot(any) != 0;
}

// a row's loss and shares from its maximum and sum, by one wave; returns the loss (all lanes)
__device__ __forceinline__ double finish_row(const LogitArgs& a, int n, float m, float s, int lane, bool& kept) {
  const float c = a.inv_t * kLog2e;
  float tt = kNegInf, ts = 0.f;
  const float log_s = log2f(s);
  const int64_t i0 = n * a.index_ld, t0 = n * a.teacher_ld;
  int64_t word;
  float t;
  for (int k = lane; k < a.K; k += 64)
    if (list_entry(a.index, i0 + k, a.wide, a.teacher, t0 + k, a.teacher_dt, word, t)) join(tt, ts, t, 1.f, c);
  join_lanes(tt, ts, 64, c);
  kept = !(ts == 0.f);  // no entry: (-inf, 0); a NaN among them: NaN
  const float tl = log2f(ts);
  float loss = 0.f;
  for (int k = lane; k < a.K; k += 64) {
    float q = 0.f, z = 0.f;
    if (list_entry(a.index, i0 + k, a.wide, a.teacher, t0 + k, a.teacher_dt, word, t)) {
      q = exp2_(fmaf(t - tt, c, -tl));
      // a word outside the vocabulary: the row's loss and gradients are NaN
      if (word >= a.V) loss = __builtin_nanf("");
      else z = load_any(a.z, n * a.z_ld + word, a.dt);
      loss += diverge(q, t, tt, tl, z, m, log_s, a.inv_t);
    }
    a.share[static_cast<int64_t>(n) * a.K + k] = q;
  }
  loss = sum_lanes(loss);
  const double all = kept ? static_cast<double>(loss) / (static_cast<double>(a.inv_t) * a.inv_t) : 0.0;
  if (lane == 0) {
    if (a.loss_each != nullptr) a.loss_each[n] = static_cast<float>(all);
    else a.rows[n] = all;
    a.top[n] = m;
    a.log_s[n] = kept ? (loss != loss ? loss : log_s) : __builtin_huge_valf();
  }
  return all;
}

// Maximum and sum of a segment; with one segment a row its loss too.  Bound by the read: 4096 x 128000
// bf16 in 195 to 232 us, 4.5 to 5.4 TB/s.  A piece's maximum first, so that an element costs one exponential.
template <int DT>
__global__ void __launch_bounds__(256) logit_stats_kernel(LogitArgs a) {
  __shared__ float red[2][4];
  typedef typename Elem<DT>::type T;
  constexpr int W = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(W))) T V;
  const int n = blockIdx.x / a.segs, seg = blockIdx.x - n * a.segs, tid = threadIdx.x, lane = tid & 63;
  const T* z = static_cast<const T*>(a.z) + n * a.z_ld;
  const int lo = seg * a.seg_len;
  int hi = lo + a.seg_len;
  if (hi > a.V) hi = a.V;
  const float c = a.inv_t * kLog2e;
  float m = kNegInf, s = 0.f;
  if (lo < hi && has_list(a, n, lane))
    walk<DT>(
        z, lo, hi, tid,
        [&](int, V v) {
          float x[W], top = m;
#pragma unroll
          for (int e = 0; e < W; ++e) {
            x[e] = to_f<DT>(v[e]);
            top = fmaxf(top, x[e]);
          }
          const float ref = top == kNegInf ? 0.f : top;
          s *= exp2_((m - ref) * c);
#pragma unroll
          for (int e = 0; e < W; ++e) s += exp2_((x[e] - ref) * c);
          m = top;
        },
        [&](int, T v) { join(m, s, to_f<DT>(v), 1.f, c); });
  join_lanes(m, s, 64, c);
  if (lane == 0) {
    red[0][tid >> 6] = m;
    red[1][tid >> 6] = s;
  }
  __syncthreads();
  if (tid < 64) {
    m = red[0][0];
    s = red[1][0];
    for (int w = 1; w < 4; ++w) join(m, s, red[0][w], red[1][w], c);
    bool kept;
    if (a.segs == 1) finish_row(a, n, m, s, lane, kept);
    else if (tid == 0) a.part[static_cast<int64_t>(n) * a.segs + seg] = make_float2(m, s);
  }
}

__device__ __forceinline__ void join_segments(const LogitArgs& a, int n, int lane, float& m, float& s) {
  const float c = a.inv_t * kLog2e;
  m = kNegInf;
  s = 0.f;
  for (int t = lane; t < a.segs; t += 64) {
    const float2 v = a.part[static_cast<int64_t>(n) * a.segs + t];
    join(m, s, v.x, v.y, c);
  }
  join_lanes(m, s, 64, c);
}

__global__ void __launch_bounds__(256) logit_finish_kernel(LogitArgs a) {
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= a.N) return;
  float m, s;
  bool kept;
  join_segments(a, n, lane, m, s);
  finish_row(a, n, m, s, lane, kept);
}

// the kept rows, and the sum or mean of their losses; with `finish` the rows' segments are joined first
__global__ void __launch_bounds__(1024) logit_reduce_kernel(LogitArgs a, int finish, float* out) {
  __shared__ double part[16];
  __shared__ int cnt[16];
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  double sum = 0.0;
  int count = 0;
  if (finish) {
    for (int n = wv; n < a.N; n += 16) {
      float m, s;
      bool kept;
      join_segments(a, n, lane, m, s);
      const double loss = finish_row(a, n, m, s, lane, kept);
      sum += loss;
      count += kept;
    }
  } else {
    for (int i = threadIdx.x; i < a.N; i += 1024) {
      sum += a.rows[i];
      count += a.log_s[i] != __builtin_huge_valf();
    }
    for (int o = 1; o < 64; o <<= 1) {
      sum += __shfl_xor(sum, o, 64);
      count += __shfl_xor(count, o, 64);
    }
  }
  if (lane == 0) {
    part[wv] = sum;
    cnt[wv] = count;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    count = 0;
    for (int w = 0; w < 16; ++w) {
      sum += part[w];
      count += cnt[w];
    }
    a.info[0] = count;
    *out = static_cast<float>(a.mean && count > 0 ? sum / count : sum);
  }
}

// The gradient: one read, one write, then the listed words of the segment once more, from the fp32
// arithmetic (a word's entries add up their shares and write the same value).  Bound by memory: 4096 x 128000
// bf16 in 430 us, 4.9 TB/s.  The last rows come first, since the forward pass has left them in the caches; a
// gradient that they cannot hold is written past them (the step of 4096 x 128000 bf16 667 -> 627 us).
template <int DT>
__global__ void __launch_bounds__(256) logit_grad_kernel(LogitArgs a) {
  constexpr int kList = 512;
  __shared__ int list_word[kList];
  __shared__ float list_share[kList];
  typedef typename Elem<DT>::type T;
  constexpr int W = 16 / sizeof(T);
  typedef __attribute__((ext_vector_type(W))) T V;
  const int n = a.N - 1 - static_cast<int>(blockIdx.x / a.segs), seg = blockIdx.x % a.segs, tid = threadIdx.x;
  const T* z = static_cast<const T*>(a.z) + n * a.z_ld;
  T* dz = static_cast<T*>(a.dz) + n * a.dz_ld;
  const int lo = seg * a.seg_len;
  int hi = lo + a.seg_len;
  if (hi > a.V) hi = a.V;
  if (lo >= hi) return;
  const float top = a.top[n], log_s = a.log_s[n], c = a.inv_t * kLog2e;
  if (log_s == __builtin_huge_valf()) {  // a row without a list: zeros, and no read
    const V none = {};
    for (int v = lo + tid * W; v < hi; v += 256 * W) {
      if (v + W <= hi) __builtin_memcpy(dz + v, &none, sizeof(V));
      else
        for (int e = v; e < hi; ++e) dz[e] = from_f<DT>(0.f);
    }
    return;
  }
  const int count = a.info[0];
  const float g = a.g[a.each ? n : 0] / a.inv_t / (a.mean && count > 0 ? static_cast<float>(count) : 1.f);
  walk<DT>(
      z, lo, hi, tid,
      [&](int v, V x) {
        V o;
#pragma unroll
        for (int e = 0; e < W; ++e) o[e] = from_f<DT>(g * exp2_(fmaf(to_f<DT>(x[e]) - top, c, -log_s)));
        if (a.stream && (reinterpret_cast<uintptr_t>(dz + v) & 15) == 0) __builtin_nontemporal_store(o, reinterpret_cast<V*>(dz + v));
        else __builtin_memcpy(dz + v, &o, sizeof(V));  // 16 bytes, of any alignment
      },
      [&](int v, T x) { dz[v] = from_f<DT>(g * exp2_(fmaf(to_f<DT>(x) - top, c, -log_s))); });
  wait_vmcnt<0>();
  __syncthreads();  // every p is written
  const int64_t i0 = n * a.index_ld;
  for (int k0 = 0; k0 < a.K; k0 += 256) {
    const int k = k0 + tid;
    const int64_t word = k < a.K ? load_index(a.index, i0 + k, a.wide) : -1;
    const bool mine = word >= lo && word < hi;
    float s = 0.f;
    for (int j0 = 0; j0 < a.K; j0 += kList) {
      const int there = a.K - j0 < kList ? a.K - j0 : kList;
      __syncthreads();
      for (int j = tid; j < there; j += 256) {
        const int64_t w = load_index(a.index, i0 + j0 + j, a.wide);
        list_word[j] = w >= lo && w < hi ? static_cast<int>(w) : -1;
        list_share[j] = a.share[static_cast<int64_t>(n) * a.K + j0 + j];
      }
      __syncthreads();
      if (mine)
        for (int j = 0; j < there; ++j) s += list_word[j] == static_cast<int>(word) ? list_share[j] : 0.f;
    }
    if (mine) dz[word] = from_f<DT>(g * (exp2_(fmaf(to_f<DT>(z[word]) - top, c, -log_s)) - s));
  }
}

// ------------------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------------------
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
int ceil_div(int64_t x, int64_t a) { return static_cast<int>((x + a - 1) / a); }

template <bool F16, int PL, bool ACOL, bool BCOL, int EPI>
int launch_gemm(hipStream_t st, const GemmArgs& a) {
  static std::atomic<uint64_t> set{0};  // the devices whose kernel has its LDS size
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e == hipSuccess && (dev > 63 || !(set.load(std::memory_order_relaxed) >> dev & 1))) {
    const void* fn = reinterpret_cast<const void*>(&gemm_kernel<F16, PL, ACOL, BCOL, EPI>);
    e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, kGemmSmem);
    if (e == hipSuccess && dev < 64) set.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  if (e != hipSuccess) return static_cast<int>(e);
  int64_t tiles = static_cast<int64_t>(ceil_div(a.M, kTile)) * ceil_div(a.N, kTile);
  tiles += 128;                                     // cut ones of the last round
  if (EPI == kPartial && tiles < 256) tiles = 256;  // pieces of the sum
  if (tiles >= (int64_t(1) << 31)) return -4;
  hipLaunchKernelGGL((gemm_kernel<F16, PL, ACOL, BCOL, EPI>), dim3(static_cast<unsigned>(tiles)), dim3(kThreads), kGemmSmem, st, a);
  return static_cast<int>(hipGetLastError());
}
template <bool ACOL, bool BCOL, int EPI>
int gemm(hipStream_t st, int dt, const GemmArgs& a) {
  if (dt == kBF16) return launch_gemm<false, 1, ACOL, BCOL, EPI>(st, a);
  if (dt == kF16) return launch_gemm<true, 1, ACOL, BCOL, EPI>(st, a);
  return launch_gemm<true, 2, ACOL, BCOL, EPI>(st, a);
}

}  // namespace

// Mirrored by vocab_loss._HeadParams.
struct DetVocabHead {
  const void *x, *w, *bias, *target, *index, *teacher;
  void *dx, *dw, *db;             // backward: null where not wanted
  const void* gout;               // backward: fp32 [1] or [N]
  float* loss;                    // forward: [1] or [N]
  void* kept;                     // what the forward pass leaves for the backward pass (Head, below)
  void* ws;
  int64_t ws_bytes, kept_bytes, x_ld, w_ld, index_ld, teacher_ld, ignore;
  int64_t hold_bytes;             // exponentials that the forward pass may hold for the backward pass (0: none follows)
  int N, D, V, K, dtype, bias_dt, wide, teacher_dt, reduction;  // reduction 0 each row, 1 mean, 2 sum
  float inv_t, smooth;
};

namespace {

// What both directions lay out in the workspace.
struct Plan {
  int planes, ldh, chunk, nchunks, parts, held, exact, twice;
  bool pack_w, keep_w, split_w, split_z, spread, again;
  int64_t off_rows_info, off_hidden, off_e, off_tops, off_kw, kept;  // in `kept`
  int64_t off_w, off_z, off_flag, off_part, off_partz, off_rows;  // forward
  int64_t off_roww, off_alpha, off_rowe, off_most, off_again, off_g, off_dx, off_dw, off_cs, off_listed, total;  // backward
};

constexpr int64_t kChunkBytes = int64_t(512) << 20;  // G of one chunk, and the packed weights of one
// Rows of G are two where both of all fit one tile of rows.  The mean square of 128 rounding errors is near its
// expectation; of one it is up to 5 times that.  A step against 128000 x 4096 bf16: 16 rows 775 us, of one each
// 757; 128 rows 1004 and 873.
constexpr int kFewRows = 128;
constexpr int64_t kKeepBytes = int64_t(4) << 30;      // packed weights that are held from forward to backward

Plan plan(const DetVocabHead& p, bool backward) {
  Plan q = {};
  q.planes = p.dtype == kF32 ? 2 : 1;
  q.ldh = static_cast<int>(up(p.D, 8));
  q.twice = p.dtype != kF32 && p.N <= kFewRows;
  q.spread = p.dtype != kBF16 && p.reduction == 0;  // rows of any weight, whose G is fp16 (weights_kernel)
  // G^T h sums over rows, so it takes them under one scale; the logits' have one each
  q.again = p.dw != nullptr && (p.dtype == kF32 || q.spread);
  // read as they are: 16-byte rows, and 256 of them within 32-bit offsets
  q.pack_w = p.dtype == kF32 || p.D % 8 != 0 || p.w_ld % 8 != 0 || (reinterpret_cast<uintptr_t>(p.w) & 15) != 0 ||
             p.w_ld > (int64_t(1) << 21);
  const int64_t w_bytes = int64_t(2) * q.planes * p.V * q.ldh, h_bytes = up((int64_t(2) * q.planes * p.N * q.ldh) << q.twice, 256);
  q.keep_w = q.pack_w && w_bytes <= kKeepBytes;
  q.off_rows_info = up(int64_t(8) * p.N * (1 + p.K), 256);
  q.off_hidden = q.off_rows_info + up(int64_t(4) * (4 + 4 * int64_t(p.N)), 256);
  auto chunks = [&](bool of_g) {
    int64_t chunk = up(p.V, kTile);
    if (of_g) {
      const int64_t fit = kChunkBytes / (int64_t(2) * q.planes * p.N) / kTile * kTile;
      if (chunk > fit) chunk = fit;
    }
    if (q.pack_w && !q.keep_w) {
      const int64_t fit = kChunkBytes / (int64_t(2) * q.planes * q.ldh) / kTile * kTile;
      if (chunk > fit) chunk = fit;
    }
    if (chunk > (1 << 20)) chunk = 1 << 20;  // 256 rows of G stay within 32-bit offsets
    if (chunk < kTile) chunk = kTile;
    return static_cast<int>(up(ceil_div(p.V, ceil_div(p.V, chunk)), kTile));  // even ones
  };
  q.chunk = chunks(backward);
  q.nchunks = ceil_div(p.V, q.chunk);
  const int gc = chunks(true);
  // Exponentials are held in fp32 for fp32 operands and with label smoothing, where G is the difference of p and
  // eps / V: near the optimum, where they are equal, 11 bits of p would be few of G's.
  q.exact = p.dtype == kF32 || p.smooth != 0.f;
  const int64_t e_bytes = (q.exact ? 4 : 2) * int64_t(p.N);  // a word's
  const int64_t held = p.hold_bytes / e_bytes / gc * gc;  // whole chunks of G
  q.held = static_cast<int>(held < up(p.V, gc) ? held : up(p.V, gc));
  q.off_e = q.off_hidden + h_bytes;
  q.off_tops = q.off_e + e_bytes * q.held;
  q.off_kw = q.off_tops + up(int64_t(4) * p.N * (q.held / 128), 256);
  q.kept = q.off_kw + (q.keep_w ? w_bytes : 0);
  q.parts = 2 * ceil_div(p.V, kTile);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += up(bytes, 256);
    return o;
  };
  // partial sums of rows x width: one for every piece of a sum of `span`, or at most 256 tiles' worth
  auto partials = [](int64_t rows, int64_t width, int64_t span, int least) {
    int64_t n = (span / least > 1 ? span / least : 1) * rows * width;
    if (n > int64_t(256) * kTile * kTile) n = int64_t(256) * kTile * kTile;
    return 4 * (n < rows * width ? rows * width : n);
  };
  q.off_w = q.pack_w && !q.keep_w ? take(int64_t(2) * q.planes * q.chunk * q.ldh) : 0;
  if (!backward) {
    q.off_flag = take(p.N);
    q.off_part = take(int64_t(8) * p.N * q.parts);
    // few tiles of a wide model, whose stages would follow each other on few CUs: 482 x 2752 x 2738 fp32 93 us, in
    // pieces 35 and 11 to join them; one row of 4096 against 32000 words 56, and 38 and 5; but a forward pass of
    // 300 x 768 x 8000 36 and in pieces 50, of 500 x 2048 x 14000 fp32 160 and 173: there their traffic costs more
    const int64_t tiles = int64_t(ceil_div(p.N, kTile)) * ceil_div(p.V, kTile);
    q.split_z = q.nchunks == 1 && p.D >= 1024 && (tiles <= 64 || (tiles <= 128 && p.N <= 64));
    q.off_z = q.split_z ? take(partials(p.N, up(p.V, kTile), q.ldh, kLogitPiece)) : 0;
    q.off_partz = p.smooth != 0.f ? take(int64_t(4) * p.N * q.parts) : 0;
    q.off_rows = take(int64_t(8) * p.N);
  } else {
    q.off_roww = take(int64_t(4) * p.N);
    q.off_alpha = take(4);
    q.off_rowe = q.spread ? take(int64_t(4) * p.N) : 0;
    q.off_most = take(4);
    q.off_again = q.again ? take(h_bytes) : 0;
    q.off_g = take((int64_t(2) * q.planes * p.N * q.chunk) << q.twice);
    q.off_dx = p.dx != nullptr ? take(partials(int64_t(p.N) << q.twice, q.ldh, q.chunk, kPiece)) : 0;
    // few tiles under many rows (8192 x 64 x 1000 bf16: 155 us for four blocks, 20 us in pieces)
    q.split_w = int64_t(ceil_div(q.chunk, kTile)) * ceil_div(p.D, kTile) <= 128 && p.N >= 1024;
    q.off_dw = p.dw != nullptr && q.split_w ? take(partials(q.chunk, q.ldh, p.N, kPiece)) : 0;
    q.off_cs = p.db != nullptr ? take(int64_t(4) * ceil_div(p.N, kTile) * q.chunk) : 0;  // G's column sums
    q.off_listed = p.db != nullptr && p.index != nullptr ? take(int64_t(8) * q.chunk) : 0;
  }
  q.total = at;
  return q;
}

int check_head(const DetVocabHead& p) {
  if (p.N < 1 || p.D < 1 || p.V < 1 || p.K < 1) return -1;
  if (p.dtype < 0 || p.dtype > 2 || p.reduction < 0 || p.reduction > 2) return -2;
  if ((p.target == nullptr) == (p.index == nullptr)) return -3;
  if (p.hold_bytes < 0) return -5;
  // offsets inside a tile are 32-bit: 256 rows of an operand, 64 rows of G
  if (p.D > (1 << 21) || p.V > (1 << 30) || p.N > (1 << 30)) return -4;
  return 0;
}

#define DET_TRY(call)             \
  do {                            \
    const int rc_ = (call);       \
    if (rc_ != 0) return rc_;     \
  } while (0)

template <int DT>
int pack(hipStream_t st, const PackArgs& a) {
  const int64_t need = (static_cast<int64_t>(a.rows) * (a.ld / 8) + 255) / 256;
  const int blocks = static_cast<int>(need < 8192 ? need : 8192);
  hipLaunchKernelGGL((pack_kernel<DT>), dim3(blocks), dim3(256), 0, st, a);
  return static_cast<int>(hipGetLastError());
}
int pack_any(hipStream_t st, int dt, const PackArgs& a) {
  if (dt == kF32) return pack<kF32>(st, a);
  return dt == kF16 && a.row_e != nullptr ? pack<kF16>(st, a) : pack<kBF16>(st, a);
}

// The call with its kept parts in place.
struct Head : DetVocabHead {
  float* stats;  // [2, N] maxima and log2 of sums, [N, K] picked logits, [N, K] shares
  int* rows;     // [4 + 4 N]: info, the list of kept rows, each row's place in it, targets, kept rows' magnitudes
  u16* hidden;   // the packed hidden states
  char* e;       // exponentials of the first q.held words' logits
  float* tops;   // their tiles' maxima
  u16* weights;  // the packed weights, if they are packed whole
  Head(const DetVocabHead& p, const Plan& q) : DetVocabHead(p) {
    char* at = static_cast<char*>(p.kept);
    stats = reinterpret_cast<float*>(at);
    rows = reinterpret_cast<int*>(at + q.off_rows_info);
    hidden = reinterpret_cast<u16*>(at + q.off_hidden);
    e = at + q.off_e;
    tops = reinterpret_cast<float*>(at + q.off_tops);
    weights = reinterpret_cast<u16*>(at + q.off_kw);
  }
};

// the kept rows, under a scale each or (absmax) one for all
int pack_hidden(hipStream_t st, const Head& p, const Plan& q, const int* absmax, const int* row_e, u16* to) {
  PackArgs a = {};
  a.src = p.x;
  a.src_ld = p.x_ld;
  a.list = p.rows + 4;
  a.count = p.rows;
  a.absmax = absmax;
  a.each = absmax == nullptr ? p.rows + 4 + int64_t(3) * p.N : nullptr;
  a.dst = to;
  a.row_e = row_e;
  a.plane = int64_t(p.N) * q.ldh;
  a.rows = p.N;
  a.cols = p.D;
  a.ld = q.ldh;
  a.twice = q.twice;
  return pack_any(st, p.dtype, a);
}

// the weight rows v0 .. v0 + nv as an operand; packs them (all: once, in the forward pass)
int weight_operand(hipStream_t st, const Head& p, const Plan& q, char* ws, int v0, int nv, bool first, Operand* w) {
  const int64_t es = p.dtype == kF32 ? 4 : 2;
  const char* src = static_cast<const char*>(p.w) + v0 * p.w_ld * es;
  if (!q.pack_w) {
    *w = Operand{reinterpret_cast<const u16*>(src), 0, p.w_ld};
    return 0;
  }
  PackArgs a = {};
  a.src = q.keep_w ? p.w : src;
  if (p.bias != nullptr) a.bias = static_cast<const char*>(p.bias) + (q.keep_w ? 0 : int64_t(v0) * (p.bias_dt == kF32 ? 4 : 2));
  a.bias_dt = p.bias_dt;
  a.src_ld = p.w_ld;
  a.absmax = p.rows + 2;
  a.dst = q.keep_w ? p.weights : reinterpret_cast<u16*>(ws + q.off_w);
  a.plane = int64_t(q.keep_w ? p.V : q.chunk) * q.ldh;
  a.rows = q.keep_w ? p.V : nv;
  a.cols = p.D;
  a.ld = q.ldh;
  *w = Operand{a.dst + (q.keep_w ? int64_t(v0) * q.ldh : 0), a.plane, q.ldh};
  return q.keep_w && !first ? 0 : pack_any(st, p.dtype, a);
}

GemmArgs logits_args(const Head& p, const Plan& q, const Operand& w, int v0, int nv) {
  GemmArgs a = {};
  a.A = Operand{p.hidden, int64_t(p.N) * q.ldh, q.ldh};
  a.B = w;
  a.m_dyn = p.rows;
  a.info = p.rows;
  a.bits = p.rows + 4 + int64_t(3) * p.N;
  a.M = p.N;
  a.N = nv;
  a.K = q.ldh;
  if (p.bias != nullptr) a.bias = static_cast<const char*>(p.bias) + int64_t(v0) * (p.bias_dt == kF32 ? 4 : 2);
  a.bias_dt = p.bias_dt;
  a.cut = 1;
  a.c = p.inv_t * kLog2e;
  a.inv_v = 1.f / static_cast<float>(p.V);
  if (p.target != nullptr) a.words = p.rows + 4 + int64_t(2) * p.N;
  a.v0 = v0;
  a.picked = p.stats + int64_t(2) * p.N;
  a.share = 1.f - p.smooth;
  a.twice = q.twice;
  return a;
}

}  // namespace

extern "C" {

// bytes of `kept` (what 0), of the forward pass's workspace (1), of the backward pass's (2)
int64_t det_vocab_head_bytes(const DetVocabHead* p, int what) {
  if (p == nullptr || check_head(*p) != 0) return -1;
  const Plan q = plan(*p, what == 2);
  return what == 0 ? q.kept : q.total;
}

int det_vocab_head_forward(void* stream, const DetVocabHead* pp) {
  if (pp == nullptr) return -1;
  DET_TRY(check_head(*pp));
  const Plan q = plan(*pp, false);
  if (pp->ws == nullptr || pp->ws_bytes < q.total || pp->kept == nullptr || pp->kept_bytes < q.kept) return -6;
  const Head p(*pp, q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(p.ws);
  int* list = p.rows + 4;

  RowArgs r = {p.target, p.index, p.teacher, reinterpret_cast<uint8_t*>(ws + q.off_flag), p.rows, list, list + p.N, list + int64_t(2) * p.N,
               p.reduction == 0 ? p.loss : nullptr, p.ignore, p.index_ld, p.teacher_ld, p.N, p.K, p.V, p.wide, p.teacher_dt};
  if (p.index != nullptr) hipLaunchKernelGGL(list_flags_kernel, dim3(ceil_div(p.N, 4)), dim3(256), 0, st, r);
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(1024), 0, st, r);
  if (p.dtype == kF32) {
    const int xb = p.N < 1024 ? ceil_div(p.N, 4) : 256, wb = p.V < 2048 ? ceil_div(p.V, 4) : 512;
    hipLaunchKernelGGL(absmax_kernel, dim3(xb + wb), dim3(256), 0, st,
                       Matrix{static_cast<const float*>(p.x), p.x_ld, p.N, p.D, list, p.rows, list + int64_t(3) * p.N, nullptr, 0},
                       Matrix{static_cast<const float*>(p.w), p.w_ld, p.V, p.D, nullptr, nullptr, nullptr, p.bias, p.bias_dt}, xb, p.rows);
  }
  DET_TRY(static_cast<int>(hipGetLastError()));
  DET_TRY(pack_hidden(st, p, q, nullptr, nullptr, p.hidden));
  for (int c = 0; c < q.nchunks; ++c) {
    const int v0 = c * q.chunk, nv = p.V - v0 < q.chunk ? p.V - v0 : q.chunk;
    Operand w;
    DET_TRY(weight_operand(st, p, q, ws, v0, nv, c == 0, &w));
    GemmArgs a = logits_args(p, q, w, v0, nv);
    a.part = reinterpret_cast<float2*>(ws + q.off_part);
    a.part_z = p.smooth != 0.f ? reinterpret_cast<float*>(ws + q.off_partz) : nullptr;
    a.parts = q.parts;
    a.E = q.held > 0 ? p.e : nullptr;
    a.tops = p.tops;
    a.held = q.held;
    a.exact = q.exact;
    if (q.split_z) {
      a.twice = 0;
      a.chunk = a.K;
      a.least = kLogitPiece;
      a.out32 = reinterpret_cast<float*>(ws + q.off_z);
      a.ldo = up(p.V, kTile);
      DET_TRY((gemm<false, false, kPartial>(st, p.dtype, a)));
      const int64_t pb = (int64_t(p.N) * ceil_div(p.V, kTile) + 3) / 4;
      hipLaunchKernelGGL(pieces_kernel, dim3(pb < 8192 ? static_cast<unsigned>(pb) : 8192u), dim3(256), 0, st, a, q.planes);
    } else {
      DET_TRY((gemm<false, false, kStats>(st, p.dtype, a)));
    }
  }
  FinishArgs f = {};
  f.x = p.x;
  f.w = p.w;
  f.bias = p.bias;
  f.x_ld = p.x_ld;
  f.w_ld = p.w_ld;
  f.dt = p.dtype;
  f.bias_dt = p.bias_dt;
  f.D = p.D;
  f.V = p.V;
  f.K = p.K;
  f.N = p.N;
  f.parts = q.parts;
  f.info = p.rows;
  f.list = list;
  f.part = reinterpret_cast<const float2*>(ws + q.off_part);
  f.part_z = p.smooth != 0.f ? reinterpret_cast<const float*>(ws + q.off_partz) : nullptr;
  f.words = list + int64_t(2) * p.N;
  f.index = p.index;
  f.teacher = p.teacher;
  f.index_ld = p.index_ld;
  f.teacher_ld = p.teacher_ld;
  f.wide = p.wide;
  f.teacher_dt = p.teacher_dt;
  f.inv_t = p.inv_t;
  f.smooth = p.smooth;
  f.top = p.stats;
  f.log_s = p.stats + p.N;
  f.picked = p.stats + int64_t(2) * p.N;
  f.share = f.picked + int64_t(p.N) * p.K;
  f.each = p.reduction == 0 ? p.loss : nullptr;
  f.rows = reinterpret_cast<double*>(ws + q.off_rows);
  if (p.target != nullptr) {
    const int blocks = ceil_div(p.N, 4);
    hipLaunchKernelGGL(finish_target_kernel, dim3(blocks < 4096 ? blocks : 4096), dim3(256), 0, st, f);
  } else {
    const dim3 fg(p.N < 8192 ? p.N : 8192);
    if (p.dtype == kF32) hipLaunchKernelGGL(finish_list_kernel<kF32>, fg, dim3(256), 0, st, f);
    else if (p.dtype == kBF16) hipLaunchKernelGGL(finish_list_kernel<kBF16>, fg, dim3(256), 0, st, f);
    else hipLaunchKernelGGL(finish_list_kernel<kF16>, fg, dim3(256), 0, st, f);
  }
  if (f.each == nullptr) hipLaunchKernelGGL(reduce_kernel, dim3(1), dim3(1024), 0, st, f.rows, p.rows, p.reduction == 1, p.loss);
  return static_cast<int>(hipGetLastError());
}

int det_vocab_head_backward(void* stream, const DetVocabHead* pp) {
  if (pp == nullptr) return -1;
  DET_TRY(check_head(*pp));
  const Plan q = plan(*pp, true);
  if (pp->ws == nullptr || pp->ws_bytes < q.total || pp->kept == nullptr || pp->kept_bytes < q.kept || pp->gout == nullptr) return -6;
  const Head p(*pp, q);
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(p.ws);
  int* list = p.rows + 4;
  const bool f16 = p.dtype != kBF16;
  const float* picked = p.stats + int64_t(2) * p.N;
  const float g_scale = f16 ? static_cast<float>(1 << kGExp) : 1.f;
  Alpha alpha = {static_cast<const float*>(p.gout), p.rows, 1.f / (p.inv_t * g_scale), p.reduction == 1};
  float* row_w = nullptr;
  int* row_e = q.spread ? reinterpret_cast<int*>(ws + q.off_rowe) : nullptr;
  u16* hidden = p.hidden;        // as G^T h takes them,
  const int* bits = p.rows + 1;  // and what their scale is made of (fp32)
  if (p.reduction == 0) {
    row_w = reinterpret_cast<float*>(ws + q.off_roww);
    float* top = reinterpret_cast<float*>(ws + q.off_alpha);
    int* most = reinterpret_cast<int*>(ws + q.off_most);
    bits = most;
    hipLaunchKernelGGL(weights_kernel, dim3(1), dim3(1024), 0, st,
                       WeightArgs{alpha.p, p.rows, list, row_w, top, row_e, p.dtype == kF32 ? list + int64_t(3) * p.N : nullptr, most, g_scale});
    DET_TRY(static_cast<int>(hipGetLastError()));
    alpha.p = top;
  }
  if (q.again) {
    hidden = reinterpret_cast<u16*>(ws + q.off_again);
    DET_TRY(pack_hidden(st, p, q, bits, row_e, hidden));
  }
  // a word's listed shares add up to N times the largest weight at most: in steps of 2^-61 N of that, below 2^63
  unsigned long long* listed = p.db != nullptr && p.index != nullptr ? reinterpret_cast<unsigned long long*>(ws + q.off_listed) : nullptr;
  double steps = 2305843009213693952.0 / g_scale;  // 2^61
  for (int64_t n = 1; n < p.N; n *= 2) steps /= 2;
  const int64_t es = p.dtype == kF32 ? 4 : 2;
  for (int c = 0; c < q.nchunks; ++c) {
    const int v0 = c * q.chunk, nv = p.V - v0 < q.chunk ? p.V - v0 : q.chunk;
    const int ldg = static_cast<int>(up(nv, 64));  // columns past nv hold -w eps / V; what they meet is fetched as zeros
    const bool held = v0 < q.held;
    Operand w = {};
    if (!held || p.dx != nullptr) DET_TRY(weight_operand(st, p, q, ws, v0, nv, false, &w));
    GemmArgs a = logits_args(p, q, w, v0, nv);
    float* cs = p.db != nullptr ? reinterpret_cast<float*>(ws + q.off_cs) : nullptr;
    a.top = p.stats;
    a.log_s = p.stats + p.N;
    a.row_w = row_w;
    a.row_e = row_e;
    a.g_scale = g_scale;
    a.smooth_v = p.smooth / static_cast<float>(p.V);
    a.colsum = cs;
    a.G = reinterpret_cast<u16*>(ws + q.off_g);
    a.g_plane = int64_t(p.N) * ldg;
    a.ldg = ldg;
    if (held) {
      const HeldArgs h = {p.e + int64_t(q.exact ? 4 : 2) * v0, p.tops + v0 / 128, q.held, p.rows, a.top, a.log_s, row_w, row_e, g_scale, a.c,
                          a.smooth_v, a.share, a.words, v0, a.colsum, a.G, a.g_plane, ldg, q.twice};
      const dim3 hg(static_cast<unsigned>(ldg / 64) * ceil_div(p.N, kTile));
      if (p.dtype == kF32) hipLaunchKernelGGL((held_kernel<kF32, true>), hg, dim3(256), 0, st, h);
      else if (p.dtype == kBF16 && q.exact) hipLaunchKernelGGL((held_kernel<kBF16, true>), hg, dim3(256), 0, st, h);
      else if (p.dtype == kBF16) hipLaunchKernelGGL((held_kernel<kBF16, false>), hg, dim3(256), 0, st, h);
      else if (q.exact) hipLaunchKernelGGL((held_kernel<kF16, true>), hg, dim3(256), 0, st, h);
      else hipLaunchKernelGGL((held_kernel<kF16, false>), hg, dim3(256), 0, st, h);
    } else {
      DET_TRY((gemm<false, false, kGrad>(st, p.dtype, a)));
    }
    if (p.index != nullptr) {
      ScatterArgs s = {p.rows, list, p.index, p.index_ld, p.wide, p.K, v0, nv, f16, q.planes, ldg, picked,
                       picked + int64_t(p.N) * p.K, a.top, a.log_s, row_w, row_e, g_scale, a.c, a.G, a.g_plane, q.twice, listed,
                       steps};
      if (listed != nullptr) hipLaunchKernelGGL(clear_kernel, dim3(ceil_div(nv, 256)), dim3(256), 0, st, listed, nv);
      const int64_t sb = (int64_t(p.N) * p.K + 255) / 256;
      hipLaunchKernelGGL(scatter_kernel, dim3(sb < 8192 ? static_cast<unsigned>(sb) : 8192u), dim3(256), 0, st, s);
    }
    const Operand G = {a.G, a.g_plane, ldg};
    if (cs != nullptr)
      hipLaunchKernelGGL(dbias_kernel, dim3(ceil_div(nv, 256)), dim3(256), 0, st, cs, ldg, nv, listed, steps, alpha, p.db, int64_t(v0),
                         p.bias_dt);
    DET_TRY(static_cast<int>(hipGetLastError()));
    if (p.dx != nullptr) {
      GemmArgs d = {};
      d.A = G;
      d.B = w;
      d.m_dyn = p.rows;
      d.info = p.rows;
      d.twice = q.twice;
      d.least = kPiece;
      d.M = p.N << q.twice;
      d.N = p.D;
      d.K = nv;
      d.chunk = q.chunk;
      d.cut = 1;
      d.out32 = reinterpret_cast<float*>(ws + q.off_dx);
      d.ldo = q.ldh;
      d.add = c > 0;
      DET_TRY((gemm<false, true, kPartial>(st, p.dtype, d)));
    }
    if (p.dw != nullptr) {
      GemmArgs d = {};
      d.A = G;
      d.B = Operand{hidden, int64_t(p.N) * q.ldh, q.ldh};
      d.k_dyn = p.rows;
      d.info = p.rows;
      d.bits = bits;
      d.twice = q.twice;
      d.least = kPiece;
      d.M = nv;
      d.N = p.D;
      d.K = p.N << q.twice;
      d.out = static_cast<char*>(p.dw) + int64_t(v0) * p.D * es;
      if (q.split_w) {
        d.out32 = reinterpret_cast<float*>(ws + q.off_dw);
        d.ldo = q.ldh;
        DET_TRY((gemm<true, true, kPartial>(st, p.dtype, d)));
        hipLaunchKernelGGL(sum_kernel, dim3(nv, ceil_div(p.D, 1024) < 64 ? ceil_div(p.D, 1024) : 64), dim3(256), 0, st, d.out32, 0,
                           d.ldo, p.rows, bits, nullptr, nullptr, 0, alpha, q.planes, d.out, p.dtype, p.D);
      } else {
        d.cut = 1;
        d.ldo = p.D;
        d.alpha = alpha;
        DET_TRY((gemm<true, true, kOut>(st, p.dtype, d)));
      }
    }
  }
  if (p.dx != nullptr)
    hipLaunchKernelGGL(sum_kernel, dim3(p.N, ceil_div(p.D, 1024) < 64 ? ceil_div(p.D, 1024) : 64), dim3(256), 0, st,
                       reinterpret_cast<const float*>(ws + q.off_dx), q.chunk, int64_t(q.ldh), p.rows, p.rows + 2, list + p.N, row_e, q.twice,
                       alpha, q.planes, p.dx, p.dtype, p.D);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"

// Mirrored by vocab_loss._LogitParams.
struct DetVocabLogits {
  const void *z, *index, *teacher;
  void* dz;
  const void* gout;
  float* loss;
  // [2, N] maxima and log2 of sums, [N, K] shares, how many rows have a list: forward writes, backward reads;
  // then the forward pass's workspace
  float* kept;
  int64_t kept_bytes, z_ld, index_ld, teacher_ld, dz_ld;
  int N, V, K, dtype, wide, teacher_dt, reduction;
  float inv_t;
};

namespace {

int64_t logit_kept(const DetVocabLogits& p) { return up(int64_t(4) * p.N * (2 + p.K) + 4, 256); }

LogitArgs logit_args(const DetVocabLogits& p) {
  LogitArgs a = {};
  a.z = p.z;
  a.z_ld = p.z_ld;
  a.dt = p.dtype;
  a.N = p.N;
  a.V = p.V;
  a.K = p.K;
  // few rows: a row is cut into segments until about eight blocks a CU run, none under 2048 long
  int64_t segs = p.N < 2048 ? 2048 / p.N : 1;
  const int64_t most = p.V / 2048 > 0 ? p.V / 2048 : 1;
  if (segs > most) segs = most;
  a.seg_len = static_cast<int>(up(ceil_div(p.V, segs), 8));
  a.segs = ceil_div(p.V, a.seg_len);
  a.index = p.index;
  a.teacher = p.teacher;
  a.index_ld = p.index_ld;
  a.teacher_ld = p.teacher_ld;
  a.wide = p.wide;
  a.teacher_dt = p.teacher_dt;
  a.inv_t = p.inv_t;
  a.each = p.reduction == 0;
  a.mean = p.reduction == 1;
  a.top = p.kept;
  a.log_s = p.kept + p.N;
  a.share = p.kept + int64_t(2) * p.N;
  a.info = reinterpret_cast<int*>(a.share + int64_t(p.N) * p.K);
  char* ws = reinterpret_cast<char*>(p.kept) + logit_kept(p);
  a.part = reinterpret_cast<float2*>(ws);
  a.rows = reinterpret_cast<double*>(ws + up(int64_t(8) * p.N * a.segs, 256));
  a.loss_each = a.each ? p.loss : nullptr;
  a.g = static_cast<const float*>(p.gout);
  a.dz = p.dz;
  a.dz_ld = p.dz_ld;
  a.stream = static_cast<int64_t>(p.N) * p.V * (p.dtype == kF32 ? 4 : 2) > (int64_t(128) << 20);
  return a;
}

int check_logits(const DetVocabLogits& p) {
  if (p.N < 1 || p.V < 1 || p.K < 1) return -1;
  if (p.dtype < 0 || p.dtype > 2 || p.reduction < 0 || p.reduction > 2) return -2;
  if (p.V > (1 << 30) || p.N > (1 << 30)) return -4;
  return 0;
}

}  // namespace

extern "C" {

int64_t det_vocab_logits_bytes(const DetVocabLogits* p) {
  if (p == nullptr || check_logits(*p) != 0) return -1;
  return logit_kept(*p) + up(int64_t(8) * p->N * logit_args(*p).segs, 256) + up(int64_t(8) * p->N, 256);
}

int det_vocab_logits_forward(void* stream, const DetVocabLogits* pp) {
  if (pp == nullptr) return -1;
  const DetVocabLogits& p = *pp;
  DET_TRY(check_logits(p));
  if (p.kept == nullptr || p.kept_bytes < det_vocab_logits_bytes(pp)) return -6;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const LogitArgs a = logit_args(p);
  const dim3 grid(static_cast<unsigned>(p.N) * a.segs);
  if (p.dtype == kF32) hipLaunchKernelGGL(logit_stats_kernel<kF32>, grid, dim3(256), 0, st, a);
  else if (p.dtype == kBF16) hipLaunchKernelGGL(logit_stats_kernel<kBF16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(logit_stats_kernel<kF16>, grid, dim3(256), 0, st, a);
  // a loss for each row needs no sum; a few rows are finished by the block that sums them
  const bool few = p.N <= 32 && !a.each;
  if (a.segs > 1 && !few) hipLaunchKernelGGL(logit_finish_kernel, dim3(ceil_div(p.N, 4)), dim3(256), 0, st, a);
  if (!a.each) hipLaunchKernelGGL(logit_reduce_kernel, dim3(1), dim3(1024), 0, st, a, a.segs > 1 && few ? 1 : 0, p.loss);
  return static_cast<int>(hipGetLastError());
}

int det_vocab_logits_backward(void* stream, const DetVocabLogits* pp) {
  if (pp == nullptr) return -1;
  const DetVocabLogits& p = *pp;
  DET_TRY(check_logits(p));
  if (p.gout == nullptr || p.dz == nullptr || p.kept == nullptr || p.kept_bytes < det_vocab_logits_bytes(pp)) return -6;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LogitArgs a = logit_args(p);
  const dim3 grid(static_cast<unsigned>(p.N) * a.segs);
  if (p.dtype == kF32) hipLaunchKernelGGL(logit_grad_kernel<kF32>, grid, dim3(256), 0, st, a);
  else if (p.dtype == kBF16) hipLaunchKernelGGL(logit_grad_kernel<kBF16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(logit_grad_kernel<kF16>, grid, dim3(256), 0, st, a);
  return static_cast<int>(hipGetLastError());
}

}  // extern "C"
