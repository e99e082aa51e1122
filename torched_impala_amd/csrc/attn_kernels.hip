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
// with in_i = e^{g(i+1)} and out_j = e^{g(L-1-j)} going forward, and the two
// exchanged going backward; each is 0 where a done lies between. Four waves
// split the value axis, so a wave's part of S never leaves its registers: in
// the layout of a matrix product's result it is already the left operand of
// the next one. Only P passes between waves, through LDS.
//
// bf16 runs on v_mfma_f32_16x16x32_bf16. What is computed in 32 bits and has
// to become an operand again is split into bf16 parts, so that the rounding
// of operands does not add to that of the result: P and S into two (2^-17,
// against 2^-9 of the bf16 result), the weighted c of the state update into
// three (2^-25), because the state is carried on in fp32. fp32 and fp16 run
// on v_mfma_f32_16x16x4_f32: the range of fp16 does not hold a state.
//
// Long sequences of few heads are cut into segments: a first pass leaves
// every segment's own state, a scan over segments turns them into entry
// states, and the segments then run side by side.
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
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int C = 64;         // steps in a chunk: one wave's ballot of dones
constexpr int THREADS = 256;

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
// --------------------------------------------------------------------------
struct EngineBF16 {
  typedef bf16_t L;              // type in LDS
  typedef bf16x8 Frag;
  static constexpr int PAD = 8;  // row padding in LDS: rows 4 banks apart
  static constexpr int NP = 2;   // parts of P and of S as operands
  static constexpr int NU = 3;   // parts of the weighted c

  static __device__ f32x4 mma(const Frag& a, const Frag& b, f32x4 acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  }
  // rows row0 + m, k along the row
  static __device__ Frag rows(const L* p, int ld, int row0, int k0, int l) {
    const L* q = p + (row0 + (l & 15)) * ld + k0 + 4 * (l >> 4);
    const bf16x4 x = *reinterpret_cast<const bf16x4*>(q);
    const bf16x4 y = *reinterpret_cast<const bf16x4*>(q + 16);
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
  static __device__ float at(const Frag& f, int e) { return (float)f[e]; }
  // a fp32 value in N bf16 parts
  template <int N>
  static __device__ void split(const float* v, Frag* out) {
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = v[e];
      #pragma unroll
      for (int n = 0; n < N; ++n) {
        const bf16_t h = (bf16_t)x;
        out[n][e] = h;
        x -= (float)h;
      }
    }
  }
  static __device__ void store4(L* p, long part, const float* v) {
    bf16x4 h, w;
    #pragma unroll
    for (int r = 0; r < 4; ++r) {
      h[r] = (bf16_t)v[r];
      w[r] = (bf16_t)(v[r] - (float)h[r]);
    }
    *reinterpret_cast<bf16x4*>(p) = h;
    *reinterpret_cast<bf16x4*>(p + part) = w;
  }
};

struct EngineF32 {
  typedef float L;
  struct Frag { f32x4 x[2]; };
  static constexpr int PAD = 4;
  static constexpr int NP = 1;
  static constexpr int NU = 1;

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
  static __device__ float at(const Frag& f, int e) { return f.x[e >> 2][e & 3]; }
  template <int N>
  static __device__ void split(const float* v, Frag* out) {
    #pragma unroll
    for (int e = 0; e < 8; ++e) out[0].x[e >> 2][e & 3] = v[e];
  }
  static __device__ void store4(L* p, long, const float* v) {
    f32x4 q = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p) = q;
  }
};

template <typename T> struct EngineOf { typedef EngineF32 E; };
template <> struct EngineOf<bf16_t> { typedef EngineBF16 E; };

// --------------------------------------------------------------------------
// one chunk's rows of one operand, in registers on the way to LDS
// --------------------------------------------------------------------------
template <typename T, int D, bool VEC>
struct Rows {
  static constexpr int V = 16 / sizeof(T);
  static constexpr int PER_ROW = D / V;
  static constexpr int N = C * PER_ROW / THREADS;
  union Piece { uint4 q; T v[V]; };
  Piece r[N];

  // rows at `p` (already at the head's first column), L of them, d columns;
  // zeros beyond
  __device__ void load(const T* p, long stride, int L, int d) {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = n * THREADS + threadIdx.x;
      const int row = idx / PER_ROW, col = (idx % PER_ROW) * V;
      r[n].q = make_uint4(0, 0, 0, 0);
      if (row < L && col < d) {
        const T* q = p + row * stride + col;
        if constexpr (VEC) {
          r[n].q = *reinterpret_cast<const uint4*>(q);
        } else {
          #pragma unroll
          for (int e = 0; e < V; ++e)
            if (col + e < d) r[n].v[e] = q[e];
        }
      }
    }
  }
  template <typename LT>
  __device__ void store(LT* s, int ld) const {
    #pragma unroll
    for (int n = 0; n < N; ++n) {
      const int idx = n * THREADS + threadIdx.x;
      const int row = idx / PER_ROW, col = (idx % PER_ROW) * V;
      LT* q = s + row * ld + col;
      if constexpr (sizeof(LT) == sizeof(T)) {
        *reinterpret_cast<uint4*>(q) = r[n].q;
      } else {   // fp16 in fp32
        #pragma unroll
        for (int e = 0; e < V; e += 4) {
          f32x4 f;
          #pragma unroll
          for (int k = 0; k < 4; ++k) f[k] = (float)r[n].v[e + k];
          *reinterpret_cast<f32x4*>(q + e) = f;
        }
      }
    }
  }
};

// --------------------------------------------------------------------------
// T: type of the operands. D: head size as it is padded, 64 or 128.
// VEC: 16-byte loads. STATE_ONLY: the first pass of cut sequences, which
// leaves a segment's own state and has no rows of a result.
// --------------------------------------------------------------------------
template <typename T, int D, bool VEC, bool STATE_ONLY>
__global__ void __launch_bounds__(THREADS)
attn_chunks(AttnArgs args) {
  typedef typename EngineOf<T>::E E;
  typedef typename E::L L;
  typedef typename E::Frag Frag;
  constexpr int LD = D + E::PAD;
  constexpr int LDP = C + E::PAD;
  constexpr int NT = D / 16;      // 16-row blocks of the state's first axis
  constexpr int NV = D / 64;      // 16-column blocks of a wave's value axis
  constexpr long PART = (long)C * LDP;

  __shared__ __align__(16) L sa[STATE_ONLY ? 1 : C * LD];
  __shared__ __align__(16) L sb[C * LD];
  __shared__ __align__(16) L sc[C * LD];
  __shared__ __align__(16) L sp[STATE_ONLY ? 1 : E::NP * C * LDP];
  __shared__ float pw[C + 1];
  __shared__ __align__(16) float w_out[C];
  __shared__ float w_in[C];
  __shared__ short2 span[C];

  const int tid = threadIdx.x;
  const int l = tid & 63, m = l & 15, g = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // blocks of one item (head and segment) in all roles go to one XCD, whose
  // L2 then holds the rows that the roles share
  const long items = (long)args.B * args.H * args.nseg;
  const int nr = args.nroles;
  const long id = blockIdx.x;
  const long full = items / 8 * 8;     // the last items % 8 are laid out plainly
  long item;
  int role_i;
  if (id < full * nr) {
    const long slot = id >> 3;
    role_i = (int)(slot % nr);
    item = (slot / nr) * 8 + (id & 7);
  } else {
    const long rest = id - full * nr;
    role_i = (int)(rest % nr);
    item = full + rest / nr;
  }
  const AttnRole& R = args.role[role_i];
  const int seg = (int)(item / ((long)args.B * args.H));
  const long bh = item % ((long)args.B * args.H);
  const int b = (int)(bh / args.H), h = (int)(bh % args.H);
  const int dk = R.dk, dv = R.dv;
  const bool rev = R.rev != 0;

  const long t_lo = seg * args.seg_len;
  const long t_hi = t_lo + args.seg_len < args.T ? t_lo + args.seg_len
                                                 : args.T;
  const int chunks = (int)((t_hi - t_lo + C - 1) / C);

  const T* pa = (const T*)R.a.p + b * R.a.sb + h * R.a.sh;
  const T* pb = (const T*)R.b.p + b * R.b.sb + h * R.b.sh;
  const T* pc = (const T*)R.c.p + b * R.c.sb + h * R.c.sh;
  T* po = (T*)R.out + ((long)b * args.H + h) * dv;
  const long so = (long)args.B * args.H * dv;
  const unsigned char* pd = args.done ? args.done + b * args.done_sb : nullptr;

  const Decay decay(args.log_decay[h * args.g_stride]);
  if (tid <= C) pw[tid] = decay.pow((float)tid);
  if constexpr (!STATE_ONLY) {
    // blocks of P that the mask leaves out and a step over 32 values of k
    // touches stay zero
    for (int i = tid; i < E::NP * C * LDP; i += THREADS) sp[i] = (L)0.f;
  }

  // the wave's part of S: block t, columns 16 (wave + 4 v) + m, rows
  // 16 t + 4 g + r
  f32x4 S[NT][NV];
  const float* s_in = R.s_in;
  bool any_state = s_in != nullptr;
  const long s_size = (long)dk * dv;
  #pragma unroll
  for (int t = 0; t < NT; ++t) {
    #pragma unroll
    for (int v = 0; v < NV; ++v) {
      S[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (any_state) {
        const int y = 16 * (wave + 4 * v) + m;
        const float* q = s_in + ((long)seg * args.B * args.H + bh) * s_size;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int x = 16 * t + 4 * g + r;
          if (x < dk && y < dv) S[t][v][r] = q[x * R.sx + y * R.sy];
        }
      }
    }
  }

  Rows<T, D, VEC> ra, rb, rc;
  int dn = 0;
  auto chunk_at = [&](int n) {
    return t_lo + (long)(rev ? chunks - 1 - n : n) * C;
  };
  auto fetch = [&](int n) {
    const long t0 = chunk_at(n);
    const int len = (int)(t_hi - t0 < C ? t_hi - t0 : C);
    if constexpr (!STATE_ONLY) ra.load(pa + t0 * R.a.st, R.a.st, len, dk);
    rb.load(pb + t0 * R.b.st, R.b.st, len, dk);
    rc.load(pc + t0 * R.c.st, R.c.st, len, dv);
    dn = (pd && l < len) ? pd[(t0 + l) * args.done_st] : 0;
  };
  fetch(0);
  bool seen_done = false;
  __syncthreads();

  // e^{g |i - j|} of a lane's places in a block, by the blocks' distance
  float wt[4][4];
  if constexpr (!STATE_ONLY) {
    #pragma unroll
    for (int d = 0; d < 4; ++d) {
      #pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int lag = m - 4 * g - r;
        const int n = 16 * d + (rev ? -lag : lag);
        wt[d][r] = pw[n < 0 ? 0 : n] * R.p_scale;
      }
    }
  }

  for (int n = 0; n < chunks; ++n) {
    const long t0 = chunk_at(n);
    const int len = (int)(t_hi - t0 < C ? t_hi - t0 : C);
    const int nt = (len + 15) >> 4;

    // ---- stage: rows to LDS, weights of the chunk's rows
    if constexpr (!STATE_ONLY) ra.store(sa, LD);
    rb.store(sb, LD);
    rc.store(sc, LD);
    const unsigned long long dones = __ballot(dn != 0);
    if (tid < C) {
      const unsigned long long upto = (2ull << tid) - 1;   // bits 0..tid
      const unsigned long long low = dones & upto, high = dones & ~upto;
      const float front = low ? 0.f : pw[tid + 1];
      const float back = (high || tid >= len) ? 0.f : pw[len - 1 - tid];
      w_in[tid] = (rev ? back : front) * R.in_scale;
      w_out[tid] = (rev ? (tid < len ? front : 0.f) : back) * R.u_scale;
      span[tid] = rev
          ? make_short2((short)tid,
                        (short)(high ? __ffsll(high) - 2 : C - 1))
          : make_short2((short)(low ? 63 - __clzll(low) : 0), (short)tid);
    }
    const float keep = dones ? 0.f : pw[len];
    seen_done |= dones != 0;
    __syncthreads();
    if (n + 1 < chunks) fetch(n + 1);

    // columns of the value axis that this wave works on
    const bool idle = 16 * wave >= dv;
    bool finite = true;

    if constexpr (!STATE_ONLY) {
      // ---- P, transposed in the products (a result's column is row i, its
      // rows are j), ten blocks over four waves
      #pragma unroll
      for (int e = 0; e < 3; ++e) {
        const int k = wave + 4 * e;
        if (k < 10) {
          const int hi = k >= 6 ? 3 : k >= 3 ? 2 : k >= 1 ? 1 : 0;
          const int lo = k - hi * (hi + 1) / 2;
          const int it = rev ? lo : hi, jt = rev ? hi : lo;
          if (hi < nt) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int s = 0; s < D / 32; ++s) {
              if (32 * s < dk)
                acc = E::mma(E::rows(sb, LD, 16 * jt, 32 * s, l),
                             E::rows(sa, LD, 16 * it, 32 * s, l), acc);
            }
            const int i = 16 * it + m;
            const short2 sp_i = span[i];
            float p[4];
            #pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = 16 * jt + 4 * g + r;
              const int d = hi - lo;
              const float w = d == 0 ? wt[0][r] : d == 1 ? wt[1][r]
                              : d == 2 ? wt[2][r] : wt[3][r];
              p[r] = (j >= sp_i.x && j <= sp_i.y) ? acc[r] * w : 0.f;
            }
            E::store4(sp + i * LDP + 16 * jt + 4 * g, PART, p);
          }
        }
      }
      __syncthreads();
    }

    f32x4 O[NV][4];
    Frag cf[2][NV];
    if (!idle) {
      if constexpr (!STATE_ONLY) {
        // ---- what came before the chunk: a S, weighted per row
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          #pragma unroll
          for (int it = 0; it < 4; ++it) O[v][it] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (any_state) {
          #pragma unroll
          for (int s = 0; s < D / 32; ++s) {
            if (32 * s < dk) {
              Frag sf[NV][E::NP];
              #pragma unroll
              for (int v = 0; v < NV; ++v) {
                float x[8];
                #pragma unroll
                for (int r = 0; r < 4; ++r) {
                  x[r] = S[2 * s][v][r];
                  x[4 + r] = S[2 * s + 1][v][r];
                }
                E::template split<E::NP>(x, sf[v]);
              }
              #pragma unroll
              for (int it = 0; it < 4; ++it) {
                if (it < nt) {
                  const Frag af = E::rows(sa, LD, 16 * it, 32 * s, l);
                  #pragma unroll
                  for (int v = 0; v < NV; ++v) {
                    #pragma unroll
                    for (int p = 0; p < E::NP; ++p)
                      O[v][it] = E::mma(sf[v][p], af, O[v][it]);
                  }
                }
              }
            }
          }
          #pragma unroll
          for (int it = 0; it < 4; ++it) {
            const float w = w_in[16 * it + m];
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              #pragma unroll
              for (int r = 0; r < 4; ++r)
                O[v][it][r] = w == 0.f ? 0.f : O[v][it][r] * w;
            }
          }
        }
      }
      // ---- c, as it is needed twice: left operand here, right one below
      #pragma unroll
      for (int s = 0; s < 2; ++s) {
        #pragma unroll
        for (int v = 0; v < NV; ++v)
          cf[s][v] = E::cols(sc, LD, 32 * s, 16 * (wave + 4 * v), l);
      }
      if constexpr (!STATE_ONLY) {
        #pragma unroll
        for (int it = 0; it < 4; ++it) {
          if (it < nt) {
            #pragma unroll
            for (int s = 0; s < 2; ++s) {
              // rows 32 s .. 32 s + 31 of j meet row block `it`?
              if (rev ? 2 * s + 1 >= it : 2 * s <= it) {
                #pragma unroll
                for (int p = 0; p < E::NP; ++p) {
                  const Frag pf =
                      E::rows(sp + p * PART, LDP, 16 * it, 32 * s, l);
                  #pragma unroll
                  for (int v = 0; v < NV; ++v)
                    O[v][it] = E::mma(cf[s][v], pf, O[v][it]);
                }
              }
            }
          }
        }
        float z = 0.f;
        #pragma unroll
        for (int v = 0; v < NV; ++v) {
          #pragma unroll
          for (int it = 0; it < 4; ++it) {
            #pragma unroll
            for (int r = 0; r < 4; ++r) z = fmaf(O[v][it][r], 0.f, z);
          }
        }
        // an input that is not finite always shows in the row that it
        // belongs to, where its own weight is not masked
        finite = !__any(z != 0.f);
        if (finite) {
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            const int y = 16 * (wave + 4 * v) + 4 * g;
            #pragma unroll
            for (int it = 0; it < 4; ++it) {
              const int i = 16 * it + m;
              if (i < len && y < dv) {
                T* q = po + (t0 + i) * so + y;
                if ((dv & 3) == 0) {
                  struct alignas(4 * sizeof(T)) { T e[4]; } w;
                  #pragma unroll
                  for (int r = 0; r < 4; ++r) w.e[r] = (T)O[v][it][r];
                  *reinterpret_cast<decltype(w)*>(q) = w;
                } else {
                  #pragma unroll
                  for (int r = 0; r < 4; ++r)
                    if (y + r < dv) q[r] = (T)O[v][it][r];
                }
              }
            }
          }
        }
      }
      // ---- the state behind the chunk
      f32x4 U[STATE_ONLY ? NT : 1][STATE_ONLY ? NV : 1];
      if (finite) {
        Frag cw[2][NV][E::NU];
        #pragma unroll
        for (int s = 0; s < 2; ++s) {
          const f32x4 w0 = *reinterpret_cast<const f32x4*>(
              w_out + 32 * s + 4 * g);
          const f32x4 w1 = *reinterpret_cast<const f32x4*>(
              w_out + 32 * s + 16 + 4 * g);
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            float x[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float w = e < 4 ? w0[e & 3] : w1[e & 3];
              x[e] = w == 0.f ? 0.f : E::at(cf[s][v], e) * w;
            }
            E::template split<E::NU>(x, cw[s][v]);
          }
        }
        #pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (16 * t < dk) {
            f32x4 acc[NV];
            #pragma unroll
            for (int v = 0; v < NV; ++v) acc[v] = f32x4{0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (32 * s < len) {
                const Frag bf = E::cols(sb, LD, 32 * s, 16 * t, l);
                #pragma unroll
                for (int v = 0; v < NV; ++v) {
                  #pragma unroll
                  for (int p = 0; p < E::NU; ++p)
                    acc[v] = E::mma(bf, cw[s][v][p], acc[v]);
                }
              }
            }
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              if constexpr (STATE_ONLY) {
                U[t][v] = acc[v];
              } else {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                  S[t][v][r] = (keep == 0.f ? 0.f : S[t][v][r] * keep) +
                               acc[v][r];
              }
            }
          } else if constexpr (STATE_ONLY) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) U[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
          }
        }
        if constexpr (STATE_ONLY) {
          float z = 0.f;
          #pragma unroll
          for (int t = 0; t < NT; ++t) {
            #pragma unroll
            for (int v = 0; v < NV; ++v) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) z = fmaf(U[t][v][r], 0.f, z);
            }
          }
          finite = !__any(z != 0.f);
          if (finite) {
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
              #pragma unroll
              for (int v = 0; v < NV; ++v) {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                  S[t][v][r] = (keep == 0.f ? 0.f : S[t][v][r] * keep) +
                               U[t][v][r];
              }
            }
          }
        }
      }
      // ---- step by step, where something is not finite
      if (!finite) {
        for (int q = 0; q < len; ++q) {
          const int i = rev ? len - 1 - q : q;
          const bool cut = (dones >> i) & 1;
          float o[NV];
          #pragma unroll
          for (int v = 0; v < NV; ++v) {
            o[v] = 0.f;
            const int y = 16 * (wave + 4 * v) + m;
            const float cy = (float)sc[i * LD + y] * R.u_scale;
            #pragma unroll
            for (int t = 0; t < NT; ++t) {
              #pragma unroll
              for (int r = 0; r < 4; ++r) {
                const int x = 16 * t + 4 * g + r;
                if (x < dk && y < dv) {
                  float s = S[t][v][r];
                  if (!rev) s = cut ? 0.f : s * pw[1];
                  s = fmaf((float)sb[i * LD + x], cy, s);
                  if constexpr (!STATE_ONLY)
                    o[v] = fmaf((float)sa[i * LD + x], s, o[v]);
                  if (rev) s = cut ? 0.f : s * pw[1];
                  S[t][v][r] = s;
                }
              }
            }
            if constexpr (!STATE_ONLY) {
              o[v] += __shfl_xor(o[v], 16, 64);
              o[v] += __shfl_xor(o[v], 32, 64);
              if (g == 0 && y < dv)
                po[(t0 + i) * so + y] = (T)(o[v] * R.in_scale);
            }
          }
        }
      }
    }
    any_state = true;
    __syncthreads();   // LDS is free for the next chunk
  }

  if (STATE_ONLY && tid == 0)
    args.keep[(long)seg * args.B * args.H + bh] =
        seen_done ? 0.f : decay.pow((float)(t_hi - t_lo));

  // the state behind the last step of this pass: a segment's own in the
  // first pass, the whole sequence's in the main one
  float* s_out = R.s_out;
  if (STATE_ONLY || (s_out && seg == (rev ? 0 : args.nseg - 1))) {
    float* q = s_out +
               (STATE_ONLY ? (long)seg * args.B * args.H + bh : bh) * s_size;
    #pragma unroll
    for (int t = 0; t < NT; ++t) {
      #pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int y = 16 * (wave + 4 * v) + m;
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int x = 16 * t + 4 * g + r;
          if (x < dk && y < dv) q[(long)x * dv + y] = S[t][v][r];
        }
      }
    }
  }
}

// own states of segments -> states that enter them, in place. first: what
// enters the first of them (in the direction of travel), or null for zero
__global__ void __launch_bounds__(256)
attn_scan(float* __restrict__ st, const float* __restrict__ keep,
          const float* __restrict__ first, long heads, long size, int nseg,
          int rev) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= heads * size) return;
  const long bh = i / size;
  float run = first ? first[i] : 0.f;
  for (int n = 0; n < nseg; ++n) {
    const long s = rev ? nseg - 1 - n : n;
    float* p = st + s * heads * size + i;
    const float own = *p, k = keep[s * heads + bh];
    *p = run;
    run = (k == 0.f ? 0.f : run * k) + own;
  }
}

// --------------------------------------------------------------------------
// one step: S' = e^g (1 - done) S + k v^T, o = scale q^T S'. Bound by reading
// and writing the state once. A block owns a head: V columns a thread,
// the rows in turns, the result added over the row groups in LDS.
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
  const long items = (long)a.B * a.H * a.nseg * a.nroles;
  if (state_only)
    hipLaunchKernelGGL((attn_chunks<T, D, VEC, true>), dim3((unsigned)items),
                       dim3(THREADS), 0, s, a);
  else
    hipLaunchKernelGGL((attn_chunks<T, D, VEC, false>), dim3((unsigned)items),
                       dim3(THREADS), 0, s, a);
}

template <typename T>
void run_t(const AttnArgs& a, int vec, bool state_only, hipStream_t s) {
  int d = 0;
  for (int i = 0; i < a.nroles; ++i) {
    d = a.role[i].dk > d ? a.role[i].dk : d;
    d = a.role[i].dv > d ? a.role[i].dv : d;
  }
  if (d <= 64) {
    if (vec) run<T, 64, true>(a, state_only, s);
    else run<T, 64, false>(a, state_only, s);
  } else {
    if (vec) run<T, 128, true>(a, state_only, s);
    else run<T, 128, false>(a, state_only, s);
  }
}

}  // namespace attn
}  // namespace impala

using namespace impala::attn;

extern "C" {

void launch_attn_chunks(int type, const AttnArgs* a, int vec, int state_only,
                        hipStream_t s) {
  if (type == 0) run_t<float>(*a, vec, state_only != 0, s);
  else if (type == 1) run_t<bf16_t>(*a, vec, state_only != 0, s);
  else run_t<f16_t>(*a, vec, state_only != 0, s);
}

void launch_attn_scan(float* st, const float* keep, const float* first,
                      long heads, long size, int nseg, int rev,
                      hipStream_t s) {
  const long n = heads * size;
  hipLaunchKernelGGL(attn_scan, dim3((unsigned)((n + 255) / 256)), dim3(256),
                     0, s, st, keep, first, heads, size, nseg, rev);
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
