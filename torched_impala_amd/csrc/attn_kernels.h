// Arguments of the linear-attention kernels (attn_kernels.hip). Strides are
// in elements; the last axis of every operand is contiguous.
#pragma once

namespace impala {
namespace attn {

struct AttnOperand {
  const void* p;
  long st, sb, sh;   // step, environment, head
};

// a, b (T, B, H, dk), c and out (T, B, H, dv); out is contiguous
struct AttnRole {
  AttnOperand a, b, c;
  void* out;
  int dk, dv;
  int rev;              // from the last step to the first
  float p_scale;        // of the products inside a chunk
  float in_scale;       // of what the state brings to a row
  float u_scale;        // of what a row adds to the state
  const float* s_in;    // state that enters, null for zero;
  long sx, sy;          //   (nseg, B * H, dk, dv), last two axes by strides
  float* s_out;         // state that leaves, contiguous, or null
};

struct AttnArgs {
  AttnRole role[3];
  int nroles;
  const float* log_decay;   // (H,)
  long g_stride;
  const unsigned char* done;   // (T, B) or null
  long done_st, done_sb;
  float* keep;              // first pass: (nseg, B * H), a segment's decay,
                            //   negative where a done lies in it
  long T, seg_len;          // seg_len a multiple of 64
  int B, H, nseg;
};

struct AttnStepArgs {
  AttnOperand q, k, v;      // (B, H, d), st unused
  void* out;
  const float* log_decay;
  long g_stride;
  const unsigned char* done;
  long done_sb;
  const float* s;           // state in, heads contiguous, environments apart
  float* d;                 // state out; may be the same memory
  long s_sb, d_sb;
  float scale;
  int B, H, dk, dv;
};

}  // namespace attn
}  // namespace impala
