// Linear attention with one decay per head, over time-major unrolls.
//
//   S_t = e^g (1 - done_t) S_{t-1} + k_t v_t^T        (dk x dv, fp32)
//   o_t = scale * q_t^T S_t
//
// One kernel serves forward and backward, because each gradient is the same
// sum with the operands in other roles (w_ts = e^{g (t-s)}, 0 across a done):
//
//   o_t  = scale sum_{s<=t} w_ts (q_t . k_s)  v_s     a=q  b=k  c=v
//   dq_t = scale sum_{s<=t} w_ts (do_t . v_s) k_s     a=do b=v  c=k
//   dk_s = scale sum_{t>=s} w_ts (v_s . do_t) q_t     a=v  b=do c=q   reversed
//   dv_s = scale sum_{t>=s} w_ts (k_s . q_t)  do_t    a=k  b=q  c=do  reversed
//
// A workgroup owns one head of one environment and walks chunks of 64 steps.
// Inside a chunk the sum is two masked products; what came before is in the
// state S (sum of weighted b c^T), which stays in registers:
//
//   P_ij = w_ij (a_i . b_j)
//   out_i = sum_j P_ij c_j + in_i a_i^T S
//   S    <- keep S + sum_j out_j b_j c_j^T
//
// with in_i = e^{g(i+1)}, out_j = e^{g(L-1-j)} for a chunk of L rows, each 0
// where a done lies between. Reversed roles read a chunk's rows backwards, so
// that they run the same code; what enters them has not decayed yet and what
// leaves has once more, in_i = e^{g i} and out_j = e^{g(L-j)}. The waves
// split the value axis, 16 columns each, so a wave's part of S never leaves
// its registers: in the layout of a matrix product's result it is already the
// left operand of the next one. Only P passes between waves, through LDS.
//
// bf16 runs on v_mfma_f32_16x16x32_bf16. What is computed in 32 bits and has
// to become an operand again is split into bf16 parts, so that the rounding
// of operands does not add to that of the result: P and S into two (2^-17,
// against 2^-9 of the bf16 result), the weighted c of the state update into
// three (2^-25), because the state is carried on in fp32. fp16 runs on
// v_mfma_f32_16x16x32_f16 at the same rate, except for P c: P does not fit the
// range of fp16, so both are split into two bf16 parts, c exactly. S and the
// weighted c are split into two fp16 parts (2^-23) after scaling each column
// by a power of two (below). fp32 runs on v_mfma_f32_16x16x4_f32.
//
// Long sequences of few heads are cut into segments: a first pass leaves
// every segment's own state, a scan over segments turns them into entry
// states, and the segments then run side by side.
//
// Bound: for heads of 64 in bf16 mostly memory (T=101, B=512, 4 heads with a
// state in and out: 44 us forward for 173 MB, which takes 31 us without any
// arithmetic); for heads of 128 the chain of LDS reads and products inside a
// chunk, with two waves a SIMD to hide it in (T=512, B=64, 8 heads: 116 us for
// 335 MB; LDS 45 %, vector units 28 %, matrix units 19 % busy). Tried there
// without gain: chunks of 32, four waves a SIMD (spills), two value blocks a
// wave, rows 8 banks apart for the transposing reads, reads ordered ahead of
// the products. fp32 is bound by its matrix rate, a sixteenth of bf16's.
//
// A product of masks lets NaN and infinities of the future or of an earlier
// episode through (0 * inf). A chunk whose result is not finite is computed
// again step by step, as the recurrence says, so that they reach exactly the
// steps that they reach there.

#include <hip/hip_runtime.h>

#include "attn_kernels.h"

namespace impala {
namespace attn {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int C = 64;         // steps in a chunk: one wave's ballot of dones
constexpr float CUT = -1.f;   // decay of a segment that a done lies in

// --------------------------------------------------------------------------
// e^{g n}: n * log2(e) * g in two floats, so that the rounding of a long
// product does not show in the exponent
// --------------------------------------------------------------------------
struct Decay {
  float hi, lo;
  __device__ explicit Decay(float g) {
    const float l2e = 1.44269504088896341f, l2e_lo = 1.92596299e-8f;
    hi = g * l2e;
    lo = fmaf(g, l2e, -hi) + g * l2e_lo;
  }
  __device__ float pow(float n) const {
    if (n == 0.f) return 1.f;
    const float x = hi * n;
    if (x < -200.f) return 0.f;   // g = -inf too
    const float r = fmaf(hi, n, -x) + lo * n;
    return exp2f(x) * fmaf(r, 0.693147181f, 1.f);
  }
};

// --------------------------------------------------------------------------
// operands of a 16 x 16 product over 32 values of k. Lane l = 16 g + m holds
// row (or column) m; its values are k = 4 g + r and 16 + 4 g + r, r = 0..3:
// two blocks of a product's result, as they come.
//
// L: type in LDS, P: type of the parts of P there. PAD: of a row in LDS, so
// that rows are 4 banks apart. NP: parts of P and of S as operands, NU: of
// the weighted c. SCALED: S and the weighted c are brought into the range of
// their parts by a power of two a column.
// --------------------------------------------------------------------------
template <typename F>
struct Frag16 {   // reads of 16-bit values
  typedef F L;
  typedef F Frag __attribute__((ext_vector_type(8)));
  typedef F Quad __attribute__((ext_vector_type(4)));
  // rows row0 + m, k along the row
  static __device__ Frag rows(const L* p, int ld, int row0, int k0, int l) {
    const L* q = p + (row0 + (l & 15)) * ld + k0 + 4 * (l >> 4);
    const Quad x = *reinterpret_cast<const Quad*>(q);
    const Quad y = *reinterpret_cast<const Quad*>(q + 16);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // columns col0 + m, k down the rows: the transposing read. In a group of
  // 16 lanes, lane 4 r + c reads 4 values of row r; lane m gets column m
  static __device__ Frag cols(const L* p, int ld, int k0, int col0, int l) {
    const int s = l & 15;
    const L* q = p + (k0 + 4 * (l >> 4) + (s >> 2)) * ld + col0 +
                 (s & 3) * 4;
    typedef __attribute__((address_space(3))) s16x4 lds_t;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_t*)const_cast<L*>(q));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_t*)const_cast<L*>(q + 16 * ld));
    return __builtin_bit_cast(
        Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  // fp32 values in N parts each, two at a time as the hardware converts
  template <int N>
  static __device__ void split(const float* v, Frag* out) {
    typedef F Two __attribute__((ext_vector_type(2)));
    #pragma unroll
    for (int e = 0; e < 8; e += 2) {
      f32x2 x = {v[e], v[e + 1]};
      #pragma unroll
      for (int n = 0; n < N; ++n) {
        const Two h = __builtin_convertvector(x, Two);
        out[n][e] = h[0];
        out[n][e + 1] = h[1];
        if (n + 1 < N) x -= __builtin_convertvector(h, f32x2);
      }
    }
  }
};

struct EngineBF16 : Frag16<bf16_t> {
  typedef bf16_t P;
  typedef Frag PFrag;
  typedef Frag CFrag;
  static constexpr int PAD = 8;
  static constexpr int NP = 2;
  static constexpr int NU = 3;
  static constexpr bool SCALED = false;

  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  }
  static __device__ CFrag c_of(const Frag& f) { return f; }
  static __device__ float at(const Frag& f, int e) { return (float)f[e]; }
  static __device__ f32x4 mma_pc(const CFrag& c, const PFrag& p, int,
                                 f32x4 acc) {
    return mma(c, p, acc);
  }
  static __device__ PFrag p_rows(const P* p, int ld, int row0, int k0,
                                 int l) {
    return rows(p, ld, row0, k0, l);
  }
  static __device__ void p_split(const float* v, PFrag* out) {
    split<NP>(v, out);
  }
  static __device__ void store4(P* p, int part, f32x4 x) {
    const bf16x4 h = __builtin_convertvector(x, bf16x4);
    *reinterpret_cast<bf16x4*>(p) = h;
    *reinterpret_cast<bf16x4*>(p + part) = __builtin_convertvector(
        x - __builtin_convertvector(h, f32x4), bf16x4);
  }
};

struct EngineF16 : Frag16<f16_t> {
  typedef EngineBF16 B;
  typedef bf16_t P;
  typedef B::Frag PFrag;
  struct CFrag { B::Frag hi, lo; };
  static constexpr int PAD = 8;
  static constexpr int NP = 2;
  static constexpr int NU = 2;
  static constexpr bool SCALED = true;

  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
  }
  static __device__ CFrag c_of(const Frag& f) {
    float v[8];
    #pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)f[e];
    B::Frag h[2];
    B::split<2>(v, h);
    return CFrag{h[0], h[1]};
  }
  static __device__ float at(const Frag& f, int e) { return (float)f[e]; }
  static __device__ f32x4 mma_pc(const CFrag& c, const PFrag& p, int part,
                                 f32x4 acc) {
    if (part == 0) acc = B::mma(c.lo, p, acc);
    return B::mma(c.hi, p, acc);
  }
  static __device__ PFrag p_rows(const P* p, int ld, int row0, int k0,
                                 int l) {
    return B::rows(p, ld, row0, k0, l);
  }
  static __device__ void p_split(const float* v, PFrag* out) {
    B::split<NP>(v, out);
  }
  static __device__ void store4(P* p, int part, f32x4 x) {
    B::store4(p, part, x);
  }
};

struct EngineF32 {
  typedef float L;
  typedef float P;
  struct Frag { f32x4 x[2]; };
  typedef Frag PFrag;
  typedef Frag CFrag;
  static constexpr int PAD = 4;
  static constexpr int NP = 1;
  static constexpr int NU = 1;
  static constexpr bool SCALED = false;

  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 acc) {
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
      #pragma unroll
      for (int r = 0; r < 4; ++r)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[h][r], b.x[h][r], acc,
                                                   0, 0, 0);
    }
    return acc;
  }
  static __device__ Frag rows(const L* p, int ld, int row0, int k0, int l) {
    const L* q = p + (row0 + (l & 15)) * ld + k0 + 4 * (l >> 4);
    Frag f;
    f.x[0] = *reinterpret_cast<const f32x4*>(q);
    f.x[1] = *reinterpret_cast<const f32x4*>(q + 16);
    return f;
  }
  static __device__ Frag cols(const L* p, int ld, int k0, int col0, int l) {
    const L* q = p + (k0 + 4 * (l >> 4)) * ld + col0 + (l & 15);
    Frag f;
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
      #pragma unroll
      for (int r = 0; r < 4; ++r) f.x[h][r] = q[(16 * h + r) * ld];
    }
    return f;
  }
  static __device__ void store4(L* p, int, f32x4 x) {
    *reinterpret_cast<f32x4*>(p) = x;
  }
  static __device__ CFrag c_of(const Frag& f) { return f; }
  static __device__ float at(const Frag& f, int e) { return f.x[e >> 2][e & 3]; }
  static __device__ f32x4 mma_pc(const CFrag& c, const PFrag& p, int,
                                 f32x4 acc) {
    return mma(c, p, acc);
  }
  static __device__ PFrag p_rows(const P* p, int ld, int row0, int k0,
                                 int l) {
    return rows(p, ld, row0, k0, l);
  }
  template <int N>
  static __device__ void split(const float* v, Frag* out) {
    #pragma unroll
    for (int e = 0; e < 8; ++e) out[0].x[e >> 2][e & 3] = v[e];
  }
  static __device__ void p_split(const float* v, PFrag* out) {
    split<1>(v, out);
  }
};

template <typename T> struct EngineOf { typedef EngineF32 E; };
template <> struct EngineOf<bf16_t> { typedef EngineBF16 E; };
template <> struct EngineOf<f16_t> { typedef EngineF16 E; };

// A power of two that brings a column's largest value to 2^14..2^15, and its
// reciprocal. Two fp16 parts then hold a value to 2^-23, down to 2^-17 of the
// column's largest; smaller ones are off by 2^-40 of that largest at most.
// (fp32 products instead, without any of this: 316 us against 146 forward for
// T=16384, B=2, 8 heads of 128.) top: the largest magnitude in this lane; a
// column's four lanes agree on it. Columns below 2^-87 are scaled as if they
// reached it. Infinities and NaN stay what they are. Only what is split is
// scaled: the other operand is as it came, and if that is one of fp16's
// subnormals, the instruction adds its products at the place of 2^-14 (32
// products of 2^-20: off by 2^-19.5 of their magnitudes' sum, else 2^-23.6).
struct Scale {
  float to, from;
  __device__ explicit Scale(float top) {
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    int e = (int)(__builtin_bit_cast(unsigned, top) >> 23);
    e = e > 40 ? e : 40;
    to = __builtin_bit_cast(float, (unsigned)(268 - e) << 23);
    from = __builtin_bit_cast(float, (unsigned)(e - 14) << 23);
  }
};

// How a workgroup divides its work: NV blocks of 16 value columns a wave, and
// whether the waves share the blocks of P through LDS or each computes all of
// them in registers. bf16, forward pass: heads of 64 (T=101, B=512, 4 heads)
// 44 us with two and all, 47 with one and shared; heads of 128 (T=512, B=64,
// 8 heads) 117 us with one and shared, 127 with two and shared, 123 with two
// and all. fp32 products are slow enough to be worth sharing.
template <typename T, int D> struct Split {
  static constexpr int NV = 1;
  static constexpr bool SHARE = true;
};
template <int D> struct Split<bf16_t, D> {
  static constexpr int NV = D > 64 ? 1 : 2;
  static constexpr bool SHARE = D > 64;
};
// fp16 has more of its own to keep in registers: with two blocks it spills
// (51 us against 49 with one, the same case; 31 against 28 for heads of 32).
template <int D> struct Split<f16_t, D> {
  static constexpr int NV = 1;
  static constexpr bool SHARE = D > 64;
};

// --------------------------------------------------------------------------
// One chunk's rows of one operand, in registers on the way to LDS. Loads take
// no branch: places beyond the rows and columns are clamped to real ones and
// cleared on the way out. (With a branch, the compiler merges its sides by
// copies that wait for the loads on the spot.)
// --------------------------------------------------------------------------
template <typename T, int D, int THREADS, bool VEC>
struct Rows {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int PER_ROW = D / V;
  static constexpr int STEP = THREADS / PER_ROW;   // rows between pieces
  static constexpr int N = C / STEP;
  union Piece { u32x4 q; T v[V]; };
  Piece r[N];
  int row, col;

  __device__ Rows() {
    row = threadIdx.x / PER_ROW;
    col = (threadIdx.x % PER_ROW) * V;
  }
  // len rows in the order of travel, d columns, p at the lowest step's row
  __device__ void load(const T* p, long stride, int len, int d, bool rev) {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
      int i = row + n * STEP;
      i = i < len ? i : len - 1;
      i = rev ? len - 1 - i : i;
      if constexpr (VEC) {   // 64 rows lie within 32 bits
        const unsigned off = (unsigned)i * (unsigned)(stride * sizeof(T)) +
                             (col < d ? col : 0) * (unsigned)sizeof(T);
        r[n].q = *reinterpret_cast<const u32x4*>(
            reinterpret_cast<const char*>(p) + off);
      } else {
        const T* q = p + i * stride;
        #pragma unroll
        for (int e = 0; e < V; ++e) r[n].v[e] = q[col + e < d ? col + e : 0];
      }
    }
  }
  __device__ void store(T* s, int ld, int len, int d) {
    if (len < C || d < D) {
      #pragma unroll
      for (int n = 0; n < N; ++n) {
        if constexpr (VEC) {
          if (row + n * STEP >= len || col >= d) r[n].q = u32x4{0, 0, 0, 0};
        } else {
          #pragma unroll
          for (int e = 0; e < V; ++e)
            if (row + n * STEP >= len || col + e >= d) r[n].v[e] = (T)0.f;
        }
      }
    }
    T* p = s + row * ld + col;
    #pragma unroll
    for (int n = 0; n < N; ++n)
      *reinterpret_cast<u32x4*>(p + n * STEP * ld) = r[n].q;
  }
};

// --------------------------------------------------------------------------
// T: type of the operands. D: head size as it is padded, 32 to 128. VEC:
// 16-byte loads. STATE_ONLY: the first pass of cut sequences, which leaves a
// segment's own state and has no rows of a result.
//
// Nothing inside a chunk branches on its length: rows and columns beyond the
// real ones are zeros in LDS and cost less than the waits between the basic
// blocks that a test of every 16 x 16 block makes.
// --------------------------------------------------------------------------
template <typename T, int D>
constexpr int threads_of() { return 4 * D / Split<T, D>::NV; }

template <typename T, int D, bool VEC, bool STATE_ONLY>
__global__ void __launch_bounds__((threads_of<T, D>()), 2)
attn_chunks(AttnArgs args) {
  typedef typename EngineOf<T>::E E;
  typedef typename E::L L;
  typedef typename E::Frag Frag;
  typedef typename E::PFrag PFrag;
  constexpr int THREADS = threads_of<T, D>();
  constexpr int NW = THREADS / 64;   // waves
  constexpr int NV = Split<T, D>::NV;   // 16-column blocks of a wave's values
  constexpr int NT = D / 16;         // 16-row blocks of the state's first axis
  constexpr int NS = D / 32;         // products over 32 of that axis
  constexpr int LD = D + E::PAD;
  constexpr int LDP = C + E::PAD;
  constexpr bool SHARE = Split<T, D>::SHARE && !STATE_ONLY;
  constexpr int PART = C * LDP;

  __shared__ __align__(16) L sa[STATE_ONLY ? 1 : C * LD];
  __shared__ __align__(16) L sb[C * LD];
  __shared__ __align__(16) L sc[C * LD];
  __shared__ __align__(16) typename E::P sp[SHARE ? E::NP * PART : 8];
  __shared__ float pw[C + 1];
  __shared__ __align__(16) float w_out[C];
  __shared__ float w_in[C];
  __shared__ int first[C];        // first row that a row still sees

  const int tid = threadIdx.x;
  const int l = tid & 63, m = l & 15, g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // blocks of one item (head and segment) in all roles go to one XCD, whose
  // L2 then holds the rows that the roles share
  const unsigned heads = args.B * args.H;
  const unsigned items = heads * args.nseg;
  const unsigned nr = args.nroles, id = blockIdx.x;
  const unsigned full = items & ~7u;   // the last few are laid out plainly
  unsigned item, role_i;
  if (id < full * nr) {
    const unsigned slot = id >> 3;
    role_i = slot % nr;
    item = (slot / nr) * 8 + (id & 7);
  } else {
    const unsigned rest = id - full * nr;
    role_i = rest % nr;
    item = full + rest / nr;
  }
  const AttnRole& R = args.role[role_i];
  const unsigned seg = item / heads, bh = item - seg * heads;
  const unsigned b = bh / args.H, h = bh - b * args.H;
  const int dk = R.dk, dv = R.dv;
  const bool rev = R.rev != 0;

  const long t_lo = seg * args.seg_len;
  const long t_hi = t_lo + args.seg_len < args.T ? t_lo + args.seg_len
                                                 : args.T;
  const int chunks = (int)((t_hi - t_lo + C - 1) / C);

  const T* pa = (const T*)R.a.p + b * R.a.sb + h * R.a.sh;
  const T* pb = (const T*)R.b.p + b * R.b.sb + h * R.b.sh;
  const T* pc = (const T*)R.c.p + b * R.c.sb + h * R.c.sh;
  T* po = (T*)R.out + (long)bh * dv;
  const long so = (long)heads * dv;
  // without flags a byte is read that is not looked at
  const bool has_done = args.done != nullptr;
  const unsigned char* pd =
      has_done ? args.done + b * args.done_sb
               : reinterpret_cast<const unsigned char*>(args.log_decay);
  const long done_st = has_done ? args.done_st : 0;

  Rows<T, D, THREADS, VEC> ra, rb, rc;
  unsigned dn = 0;   // as loaded: a test here would wait for all loads
  // Chunks in the order of travel, each by its lowest step. Where the next
  // one lies is carried along: the strides stay in few scalar registers.
  const int tail = (int)(t_hi - t_lo - (long)(chunks - 1) * C);
  const int tail_at = rev ? 0 : chunks - 1;
  long t_next = t_lo + (rev ? (long)(chunks - 1) * C : 0);
  const long dir = rev ? -C : C;
  const T* na = pa + t_next * R.a.st;
  const T* nb = pb + t_next * R.b.st;
  const T* nc = pc + t_next * R.c.st;
  const unsigned char* nd = pd + t_next * done_st;
  const long sta = R.a.st, stb = R.b.st, stc = R.c.st;
  // behind the last chunk one row of it is read again and not used
  auto fetch = [&](int n) __attribute__((always_inline)) {
    const int len = n >= chunks ? 1 : n == tail_at ? tail : C;
    dn = nd[(l < len ? l : len - 1) * (int)done_st];
    if constexpr (!STATE_ONLY) ra.load(na, sta, len, dk, rev);
    rb.load(nb, stb, len, dk, rev);
    rc.load(nc, stc, len, dv, rev);
    if (n + 1 < chunks) {
      na += dir * sta;
      nb += dir * stb;
      nc += dir * stc;
      nd += dir * done_st;
    }
  };
  fetch(0);

  // the wave's part of S: block t, column y0 + 16 v, rows 16 t + 4 g + r
  f32x4 S[NT][NV];
  const int y0 = 16 * NV * wave + m;
  const bool whole = dk == D && dv == D;
  const long s_size = (long)dk * dv;
  bool any_state = R.s_in != nullptr;
  #pragma unroll
  for (int t = 0; t < NT; ++t) {
    #pragma unroll
    for (int v = 0; v < NV; ++v) S[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (any_state) {
    const float* q = R.s_in + ((long)seg * heads + bh) * s_size;
    const int sx = (int)R.sx, sy = (int)R.sy;
    if (whole) {
      const unsigned at = 4 * g * sx + y0 * sy;
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          #pragma unroll
          for (int r = 0; r < 4; ++r)
            S[t][v][r] = (q + (16 * t + r) * sx + 16 * v * sy)[at];
        }
      }
    } else {   // from clamped places, all at once, and cleared beyond the size
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int y = y0 + 16 * v;
          #pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int x = 16 * t + 4 * g + r;
            S[t][v][r] = q[(x < dk ? x : dk - 1) * sx +
                           (y < dv ? y : dv - 1) * sy];
          }
        }
      }
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          #pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * t + 4 * g + r >= dk || y0 + 16 * v >= dv)
              S[t][v][r] = 0.f;
        }
      }
    }
  }

  const Decay decay(args.log_decay[h * args.g_stride]);
  for (int i = tid; i <= C; i += THREADS) pw[i] = decay.pow((float)i);
  if constexpr (SHARE) {   // blocks of P that the mask leaves out stay zero
    u32x4* z = reinterpret_cast<u32x4*>(sp);
    constexpr int NZ = E::NP * PART * (int)sizeof(typename E::P) / 16;
    for (int i = tid; i < NZ; i += THREADS) z[i] = u32x4{0, 0, 0, 0};
  }
  bool seen_done = false;
  __syncthreads();
  // a decay above zero whose powers overflow: zeros times those are NaN, so
  // such a head goes step by step too
  const bool grows = !(pw[C] <= 3.4e38f);

  // Blocks of P on and under the diagonal: with SHARE the wave's own of the
  // ten, else the four distances from it. e^{g (i - j)} at the lane's places
  // in them, 0 above the diagonal
  constexpr int NP = SHARE ? (10 + NW - 1) / NW : 4;
  float wt[NP][4];
  int p_it[NP], p_jt[NP];
  if constexpr (!STATE_ONLY) {
    #pragma unroll
    for (int e = 0; e < NP; ++e) {
      if constexpr (SHARE) {
        // a wave without a block of its own computes the last one too
        const int k = wave + NW * e < 10 ? wave + NW * e : 9;
        p_it[e] = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0;
        p_jt[e] = k - p_it[e] * (p_it[e] + 1) / 2;
      } else {
        p_it[e] = e;
        p_jt[e] = 0;
      }
      #pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int lag = 16 * (p_it[e] - p_jt[e]) + m - 4 * g - r;
        wt[e][r] = lag < 0 ? 0.f : pw[lag > C ? C : lag] * R.p_scale;
      }
    }
  }
  // this wave has columns of the result
  const bool idle = 16 * NV * wave >= dv;

  for (int n = 0; n < chunks; ++n) {
    const long t0 = t_next;
    const int len = n == tail_at ? tail : C;
    t_next += dir;

    // ---- stage: rows to LDS, weights of the chunk's rows
    if constexpr (!STATE_ONLY) ra.store(sa, LD, len, dk);
    rb.store(sb, LD, len, dk);
    rc.store(sc, LD, len, dv);
    // cuts between rows in the order of travel: bit i lies before row i. A
    // done lies before its step, so backwards one row further on, and that
    // of the lowest step behind the chunk
    unsigned long long cuts = __ballot(has_done && dn != 0 && l < len);
    const bool any_cut = cuts != 0;
    bool cut_behind = false;
    if (rev && any_cut) {
      cut_behind = cuts & 1;
      cuts = len > 1 ? __brevll(cuts >> 1) >> (C - len) : 0;
    }
    if (tid < C) {
      const unsigned long long upto = (2ull << tid) - 1;   // bits 0..tid
      const unsigned long long low = cuts & upto, high = cuts & ~upto;
      const int in = rev ? tid : tid + 1, out = rev ? len - tid : len - 1 - tid;
      w_in[tid] = low ? 0.f : pw[in] * R.in_scale;
      w_out[tid] = high || cut_behind || tid >= len ? 0.f
                                                    : pw[out] * R.u_scale;
      first[tid] = low ? 63 - __clzll(low) : 0;
    }
    const float keep = any_cut ? 0.f : pw[len];
    seen_done |= any_cut;
    __syncthreads();
    fetch(n + 1);

    bool finite = true;
    if constexpr (SHARE) {
      // ---- P, transposed in the products (a result's column is row i, its
      // rows are j)
      f32x4 acc[NP];
      #pragma unroll
      for (int e = 0; e < NP; ++e) acc[e] = f32x4{0.f, 0.f, 0.f, 0.f};
      #pragma unroll
      for (int s = 0; s < NS; ++s) {
        #pragma unroll
        for (int e = 0; e < NP; ++e)
          acc[e] = E::mma(E::rows(sb, LD, 16 * p_jt[e], 32 * s, l),
                          E::rows(sa, LD, 16 * p_it[e], 32 * s, l), acc[e]);
      }
      #pragma unroll
      for (int e = 0; e < NP; ++e) {
        #pragma unroll
        for (int r = 0; r < 4; ++r) acc[e][r] *= wt[e][r];
      }
      if (any_cut) {
        asm volatile("");   // a branch: most chunks have no cut
        #pragma unroll
        for (int e = 0; e < NP; ++e) {
          const int lo = first[16 * p_it[e] + m] - 16 * p_jt[e] - 4 * g;
          #pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < lo) acc[e][r] = 0.f;
        }
      }
      #pragma unroll
      for (int e = 0; e < NP; ++e)
        E::store4(sp + (16 * p_it[e] + m) * LDP + 16 * p_jt[e] + 4 * g, PART,
                  acc[e]);
    }

    f32x4 O[4][NV];
    Frag cf[2][NV];
    if (!idle) {
      if constexpr (!STATE_ONLY) {
        // ---- what came before the chunk: a S, weighted per row
        #pragma unroll
        for (int it = 0; it < 4; ++it) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) O[it][v] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (any_state) {
          float to[NV], back[NV][4];   // of S: a column is a row of O
          if constexpr (E::SCALED) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              float top = 0.f;
              #pragma unroll
              for (int t = 0; t < NT; ++t) {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                  top = fmaxf(top, fabsf(S[t][v][r]));
              }
              const Scale scale(top);
              to[v] = scale.to;
              #pragma unroll
              for (int r = 0; r < 4; ++r)
                back[v][r] = __shfl(scale.from, 4 * g + r, 64);
            }
          }
          #pragma unroll
          for (int s = 0; s < NS; ++s) {
            Frag sf[NV][E::NP];
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              float x[8];
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                x[r] = S[2 * s][v][r];
                x[4 + r] = S[2 * s + 1][v][r];
                if constexpr (E::SCALED) {
                  x[r] *= to[v];
                  x[4 + r] *= to[v];
                }
              }
              E::template split<E::NP>(x, sf[v]);
            }
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
              const Frag af = E::rows(sa, LD, 16 * it, 32 * s, l);
              #pragma unroll
              for (int p = 0; p < E::NP; ++p) {
                #pragma unroll
                for (int v = 0; v < NV; ++v)
                  O[it][v] = E::mma(sf[v][p], af, O[it][v]);
              }
            }
          }
          #pragma unroll
          for (int it = 0; it < 4; ++it) {
            const float w = w_in[16 * it + m];
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                if constexpr (E::SCALED) O[it][v][r] *= back[v][r];
                O[it][v][r] *= w;
              }
            }
          }
        }
      }
      // ---- c, as it is needed twice: left operand here, right one below
      #pragma unroll
      for (int s = 0; s < 2; ++s) {
        #pragma unroll
        for (int v = 0; v < NV; ++v)
          cf[s][v] = E::cols(sc, LD, 32 * s, 16 * (NV * wave + v), l);
      }
    }
    if constexpr (SHARE) __syncthreads();   // P is whole
    if (!idle) {
      if constexpr (!STATE_ONLY) {
        typename E::CFrag cc[2][NV];
        #pragma unroll
        for (int s = 0; s < 2; ++s) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) cc[s][v] = E::c_of(cf[s][v]);
        }
        // row blocks 0 and 1 meet the first 32 rows of j, 2 and 3 all
        #pragma unroll
        for (int it = 0; it < 4; ++it) {
          if constexpr (SHARE) {
            #pragma unroll
            for (int s = 0; s <= it >> 1; ++s) {
              #pragma unroll
              for (int p = 0; p < E::NP; ++p) {
                const PFrag pf =
                    E::p_rows(sp + p * PART, LDP, 16 * it, 32 * s, l);
                #pragma unroll
                for (int v = 0; v < NV; ++v)
                  O[it][v] = E::mma_pc(cc[s][v], pf, p, O[it][v]);
              }
            }
          } else {
            // ---- the row block of P, transposed in the products, so that
            // it comes out as the right operand of the next one
            f32x4 acc[4];
            #pragma unroll
            for (int jt = 0; jt < 4; ++jt) acc[jt] = f32x4{0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int s = 0; s < NS; ++s) {
              const Frag af = E::rows(sa, LD, 16 * it, 32 * s, l);
              #pragma unroll
              for (int jt = 0; jt <= it; ++jt)
                acc[jt] = E::mma(E::rows(sb, LD, 16 * jt, 32 * s, l), af,
                                 acc[jt]);
            }
            #pragma unroll
            for (int jt = 0; jt <= it; ++jt) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) acc[jt][r] *= wt[it - jt][r];
            }
            if (any_cut) {
              asm volatile("");   // a branch: most chunks have no cut
              const int lo = first[16 * it + m] - 4 * g;
              #pragma unroll
              for (int jt = 0; jt <= it; ++jt) {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (16 * jt + r < lo) acc[jt][r] = 0.f;
              }
            }
            #pragma unroll
            for (int s = 0; s <= it >> 1; ++s) {
              float x[8];
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                x[r] = acc[2 * s][r];
                x[4 + r] = acc[2 * s + 1][r];
              }
              PFrag pf[E::NP];
              E::p_split(x, pf);
              #pragma unroll
              for (int p = 0; p < E::NP; ++p) {
                #pragma unroll
                for (int v = 0; v < NV; ++v)
                  O[it][v] = E::mma_pc(cc[s][v], pf[p], p, O[it][v]);
              }
            }
          }
        }
        // An input that is not finite always shows in the row that it
        // belongs to, where its own weight is not zero; a state that is not
        // shows in every row, as weights of zero make NaN of it.
        f32x4 z = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int it = 0; it < 4; ++it) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            #pragma unroll
            for (int r = 0; r < 4; ++r) z[r] = fmaf(O[it][v][r], 0.f, z[r]);
          }
        }
        finite = !__any(grows || (z[0] + z[1]) + (z[2] + z[3]) != 0.f);
        if (finite) {
          const int x0 = 16 * NV * wave + 4 * g;
          if constexpr (VEC) {   // dv is a multiple of 4, 64 rows in 32 bits
            T* q = po + (rev ? t0 + len - C : t0) * so;
            const long step = (rev ? -16 : 16) * so;
            const unsigned at = (unsigned)((rev ? C - 1 - m : m) * so + x0);
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
              #pragma unroll
              for (int v = 0; v < NV; ++v) {
                struct alignas(4 * sizeof(T)) { T e[4]; } w;
                #pragma unroll
                for (int r = 0; r < 4; ++r) w.e[r] = (T)O[it][v][r];
                if (16 * it + m < len && x0 + 16 * v < dv)
                  *reinterpret_cast<decltype(w)*>(q + it * step + 16 * v +
                                                  at) = w;
              }
            }
          } else {
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
              const int i = 16 * it + m;
              T* q = po + (t0 + (rev ? len - 1 - i : i)) * so + x0;
              #pragma unroll
              for (int v = 0; v < NV; ++v) {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (i < len && x0 + 16 * v + r < dv)
                    q[16 * v + r] = (T)O[it][v][r];
              }
            }
          }
        }
      }
      // ---- the state behind the chunk
      if (finite) {
        f32x4 U[NT][NV];
        #pragma unroll
        for (int t = 0; t < NT; ++t) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            #pragma unroll
            for (int r = 0; r < 4; ++r)
              U[t][v][r] = E::SCALED ? 0.f : S[t][v][r] * keep;
          }
        }
        float to[NV], from[NV];   // of the weighted c
        if constexpr (E::SCALED) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            float top = 0.f;
            #pragma unroll
            for (int e = 0; e < 16; ++e)
              top = fmaxf(top, fabsf(E::at(cf[e >> 3][v], e & 7) *
                                     w_out[32 * (e >> 3) + 16 * (e >> 2 & 1) +
                                           4 * g + (e & 3)]));
            const Scale scale(top);
            to[v] = scale.to;
            from[v] = scale.from;
          }
        }
        #pragma unroll
        for (int s = 0; s < 2; ++s) {
          const f32x4 w0 = *reinterpret_cast<const f32x4*>(
              w_out + 32 * s + 4 * g);
          const f32x4 w1 = *reinterpret_cast<const f32x4*>(
              w_out + 32 * s + 16 + 4 * g);
          Frag cw[NV][E::NU];
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            float x[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float w = e < 4 ? w0[e & 3] : w1[e & 3];
              // weighted first: a zero stays one under any scale
              x[e] = E::at(cf[s][v], e) * w;
              if constexpr (E::SCALED) x[e] *= to[v];
            }
            E::template split<E::NU>(x, cw[v]);
          }
          #pragma unroll
          for (int t = 0; t < NT; ++t) {
            const Frag bf = E::cols(sb, LD, 32 * s, 16 * t, l);
            #pragma unroll
            for (int p = 0; p < E::NU; ++p) {
              #pragma unroll
              for (int v = 0; v < NV; ++v)
                U[t][v] = E::mma(bf, cw[v][p], U[t][v]);
            }
          }
        }
        if constexpr (E::SCALED) {
          #pragma unroll
          for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              #pragma unroll
              for (int r = 0; r < 4; ++r)
                U[t][v][r] = fmaf(U[t][v][r], from[v], S[t][v][r] * keep);
            }
          }
        }
        if constexpr (STATE_ONLY) {   // no rows that would show it
          f32x4 z = {0.f, 0.f, 0.f, 0.f};
          #pragma unroll
          for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) z[r] = fmaf(U[t][v][r], 0.f, z[r]);
            }
          }
          finite = !__any(grows || (z[0] + z[1]) + (z[2] + z[3]) != 0.f);
        }
        if (finite) {
          #pragma unroll
          for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) S[t][v] = U[t][v];
          }
        }
      }
      // ---- step by step, where something is not finite
      if (!finite) {
        // sizes that the compiler cannot take for those outside: it would
        // compute the masks below in front of the loop, for every chunk
        int dk_ = dk, dv_ = dv;
        asm volatile("" : "+s"(dk_), "+s"(dv_));
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int y = y0 + 16 * v;
          for (int i = 0; i < len; ++i) {
            // what lies before the first row backwards has not decayed
            const bool cut = (cuts >> i) & 1;
            const float f = rev && i == 0 ? 1.f : pw[1];
            const float cy = (float)sc[i * LD + y] * R.u_scale;
            float o = 0.f;
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int x = 16 * t + 4 * g + r;
                if (x < dk_ && y < dv_) {
                  S[t][v][r] = fmaf((float)sb[i * LD + x], cy,
                                    cut ? 0.f : S[t][v][r] * f);
                  if constexpr (!STATE_ONLY)
                    o = fmaf((float)sa[i * LD + x], S[t][v][r], o);
                }
              }
            }
            if constexpr (!STATE_ONLY) {
              o += __shfl_xor(o, 16, 64);
              o += __shfl_xor(o, 32, 64);
              if (g == 0 && y < dv_)
                po[(t0 + (rev ? len - 1 - i : i)) * so + y] =
                    (T)(o * R.in_scale);
            }
          }
          if (rev) {
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
              #pragma unroll
              for (int r = 0; r < 4; ++r)
                S[t][v][r] = cut_behind ? 0.f : S[t][v][r] * pw[1];
            }
          }
        }
      }
    }
    any_state = true;
    if (n + 1 < chunks) __syncthreads();   // LDS is free for the next chunk
  }

  // a done is not a decay of zero, which many steps without one may reach
  if (STATE_ONLY && tid == 0)
    args.keep[seg * heads + bh] =
        seen_done ? CUT : decay.pow((float)(t_hi - t_lo));

  // the state behind the last step of this pass: a segment's own in the
  // first pass, the whole sequence's in the main one
  if (STATE_ONLY || (R.s_out && (int)seg == (rev ? 0 : args.nseg - 1))) {
    float* q = R.s_out + (STATE_ONLY ? (long)seg * heads + bh : (long)bh) *
                             s_size;
    if (whole) {
      const unsigned at = 4 * g * D + y0;
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          #pragma unroll
          for (int r = 0; r < 4; ++r)
            (q + (16 * t + r) * D + 16 * v)[at] = S[t][v][r];
        }
      }
    } else {
      #pragma unroll
      for (int t = 0; t < NT; ++t) {
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int y = y0 + 16 * v;
          #pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int x = 16 * t + 4 * g + r;
            if (x < dk && y < dv) q[x * dv + y] = S[t][v][r];
          }
        }
      }
    }
  }
}

// What n steps of a segment leave of a state where it or their decay is not
// finite. The decay of them all may be zero in 32 bits, or infinite, where that
// of a step is not: what becomes of a state that is not finite is then said by
// a step, and of any other by all of them.
__device__ __attribute__((noinline)) float carry_steps(float run, float keep,
                                                       float log_decay,
                                                       long n) {
  if (keep == CUT) return 0.f;
  const float step = Decay(log_decay).pow(1.f);
  if (!isfinite(run)) return run * step;
  for (long i = 0; i < n && isfinite(run); ++i) {
    run *= step;
    if (run == 0.f) break;
  }
  return run;
}

// own states of segments -> states that enter them, in place. first: what
// enters the first of them (in the direction of travel), or null for zero
__global__ void __launch_bounds__(256)
attn_scan(float* __restrict__ st, const float* __restrict__ keep,
          const float* __restrict__ first, const float* __restrict__ log_decay,
          long g_stride, int H, long heads, long size, int nseg, int rev,
          long T, long seg_len) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= heads * size) return;
  const long bh = i / size;
  float run = first ? first[i] : 0.f;
  // eight segments are read before the first is written: a load does not move
  // over a store to the same array by itself
  for (int n0 = 0; n0 < nseg; n0 += 8) {
    float own[8], k[8];
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int n = n0 + e < nseg ? n0 + e : nseg - 1;
      const long s = rev ? nseg - 1 - n : n;
      own[e] = st[s * heads * size + i];
      k[e] = keep[s * heads + bh];
    }
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (n0 + e < nseg) {
        const long s = rev ? nseg - 1 - n0 - e : n0 + e;
        st[s * heads * size + i] = run;
        if (isfinite(run) && k[e] <= 3.4e38f) {
          run *= fmaxf(k[e], 0.f);
        } else {
          const long left = T - s * seg_len;
          run = carry_steps(run, k[e], log_decay[bh % H * g_stride],
                            left < seg_len ? left : seg_len);
        }
        run += own[e];
      }
    }
  }
}

// --------------------------------------------------------------------------
// one step: S' = e^g (1 - done) S + k v^T, o = scale q^T S'. Bound by reading
// and writing the state once: 103 us for 512 environments of 8 heads of
// 128 x 128, 5.2 TB/s, as fast as a copy; 4.4 us for 32 of 4 heads of 64 x 64,
// a launch. A block owns a head: V columns a thread, the rows in turns, the
// result added over the row groups in LDS.
// --------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(256)
attn_step(AttnStepArgs A) {
  __shared__ float sq[128], sk[128];
  __shared__ __align__(16) float so[256 * V];
  const long bh = blockIdx.x;
  const int b = (int)(bh / A.H), h = (int)(bh % A.H);
  const int tid = threadIdx.x;
  const T* q = (const T*)A.q.p + b * A.q.sb + h * A.q.sh;
  const T* k = (const T*)A.k.p + b * A.k.sb + h * A.k.sh;
  const T* v = (const T*)A.v.p + b * A.v.sb + h * A.v.sh;
  const bool cut = A.done && A.done[b * A.done_sb];
  const float lam =
      cut ? 0.f : Decay(A.log_decay[h * A.g_stride]).pow(1.f);

  const int cols = (A.dv + V - 1) / V;          // threads along a row
  int tx = 1;
  while (tx < cols) tx <<= 1;                   // <= 128
  const int ty = 256 / tx;
  const int x = tid & (tx - 1), y = tid / tx;
  const int c = x * V;
  const float* s = A.s + b * A.s_sb + h * (long)A.dk * A.dv;
  float* d = A.d + b * A.d_sb + h * (long)A.dk * A.dv;

  if (tid < A.dk) {
    sq[tid] = (float)q[tid];
    sk[tid] = (float)k[tid];
  }
  float vv[V], o[V];
  #pragma unroll
  for (int e = 0; e < V; ++e) {
    vv[e] = c + e < A.dv ? (float)v[c + e] : 0.f;
    o[e] = 0.f;
  }
  __syncthreads();
  // four rows are read before the first is written: the two states may be
  // one, so the compiler does not move a load over a store by itself
  if (c < A.dv) {
    for (int r0 = y; r0 < A.dk; r0 += 4 * ty) {
      float w[4][V];
      #pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = r0 + n * ty;
        #pragma unroll
        for (int e = 0; e < V; ++e) w[n][e] = 0.f;
        if (r < A.dk) {
          const float* p = s + (long)r * A.dv + c;
          if constexpr (V == 4) {
            const f32x4 f = *reinterpret_cast<const f32x4*>(p);
            #pragma unroll
            for (int e = 0; e < V; ++e) w[n][e] = f[e];
          } else {
            w[n][0] = *p;
          }
        }
      }
      #pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int r = r0 + n * ty;
        if (r < A.dk) {
          const float kr = sk[r], qr = sq[r];
          #pragma unroll
          for (int e = 0; e < V; ++e) {
            w[n][e] = fmaf(kr, vv[e], cut ? 0.f : w[n][e] * lam);
            o[e] = fmaf(qr, w[n][e], o[e]);
          }
          float* p = d + (long)r * A.dv + c;
          if constexpr (V == 4) {
            const f32x4 f = {w[n][0], w[n][1], w[n][2], w[n][3]};
            *reinterpret_cast<f32x4*>(p) = f;
          } else {
            *p = w[n][0];
          }
        }
      }
    }
  }
  #pragma unroll
  for (int e = 0; e < V; ++e) so[(y * tx + x) * V + e] = o[e];
  __syncthreads();
  T* out = (T*)A.out + bh * A.dv;
  for (int e = tid; e < A.dv; e += 256) {
    float sum = 0.f;
    for (int r = 0; r < ty; ++r) sum += so[r * tx * V + e];
    out[e] = (T)(sum * A.scale);
  }
}

template <typename T, int D, bool VEC>
void run(const AttnArgs& a, bool state_only, hipStream_t s) {
  const dim3 grid((unsigned)((long)a.B * a.H * a.nseg * a.nroles));
  if (state_only)
    hipLaunchKernelGGL((attn_chunks<T, D, VEC, true>), grid,
                       dim3(threads_of<T, D>()), 0, s, a);
  else
    hipLaunchKernelGGL((attn_chunks<T, D, VEC, false>), grid,
                       dim3(threads_of<T, D>()), 0, s, a);
}

template <typename T, bool VEC>
void run_t(const AttnArgs& a, bool state_only, hipStream_t s) {
  int d = 0;
  for (int i = 0; i < a.nroles; ++i) {
    d = a.role[i].dk > d ? a.role[i].dk : d;
    d = a.role[i].dv > d ? a.role[i].dv : d;
  }
  if (d <= 32) run<T, 32, VEC>(a, state_only, s);
  else if (d <= 64) run<T, 64, VEC>(a, state_only, s);
  else if (d <= 96) run<T, 96, VEC>(a, state_only, s);
  else run<T, 128, VEC>(a, state_only, s);
}

template <typename T>
void run_v(const AttnArgs& a, int vec, bool state_only, hipStream_t s) {
  if (vec) run_t<T, true>(a, state_only, s);
  else run_t<T, false>(a, state_only, s);
}

}  // namespace attn
}  // namespace impala

using namespace impala::attn;

extern "C" {

void launch_attn_chunks(int type, const AttnArgs* a, int vec, int state_only,
                        hipStream_t s) {
  if (type == 0) run_v<float>(*a, vec, state_only != 0, s);
  else if (type == 1) run_v<bf16_t>(*a, vec, state_only != 0, s);
  else run_v<f16_t>(*a, vec, state_only != 0, s);
}

void launch_attn_scan(float* st, const float* keep, const float* first,
                      const float* log_decay, long g_stride, int H,
                      long heads, long size, int nseg, int rev, long T,
                      long seg_len, hipStream_t s) {
  const long n = heads * size;
  hipLaunchKernelGGL(attn_scan, dim3((unsigned)((n + 255) / 256)), dim3(256),
                     0, s, st, keep, first, log_decay, g_stride, H, heads,
                     size, nseg, rev, T, seg_len);
}

void launch_attn_step(int type, const AttnStepArgs* a, int vec,
                      hipStream_t s) {
  const dim3 grid((unsigned)((long)a->B * a->H)), block(256);
#define IMPALA_STEP(T)                                                     \
  if (vec) hipLaunchKernelGGL((attn_step<T, 4>), grid, block, 0, s, *a);   \
  else hipLaunchKernelGGL((attn_step<T, 1>), grid, block, 0, s, *a)
  if (type == 0) { IMPALA_STEP(float); }
  else if (type == 1) { IMPALA_STEP(bf16_t); }
  else { IMPALA_STEP(f16_t); }
#undef IMPALA_STEP
}

}  // extern "C"
