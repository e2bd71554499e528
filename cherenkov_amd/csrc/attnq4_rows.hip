// Attention over the 4-bit cache for sequences with many (row, head) pairs:
// prompts, turns, documents (k_attn_q4_rows, attnq4_many.h).
//
// Rows are plenty here, so what bounds the other kernel (attnq4.hip), the
// vector work of every wave on every tile's codes, scales and least values, is
// done once for 64 or 128 rows: the workgroup turns a step's codes into f16
// operands in LDS, and its four waves, 16 RB rows each, read them.  s (c - 8)
// has 8 + 3 significant bits, f16's 11, and is scaled by a power of two of the
// token that brings the largest of its groups' 8 s and |b + 8 s| under 2^15 (of
// keys 2^12).  So an operand is exact while its group's step is above 2^-28 of
// that (of keys 2^-25), the smallest with 11 bits above f16's least 2^-24 when
// odd codes take it 16-fold smaller; further down it is off by 2^-32 of that at
// most (of keys 2^-29).  Then
//   score_t = 2^e_t ( sum_d q_d [s (c - 8)]_td + sum_g Q_g [b + 8 s]_tg )
//   out_d   = sum_t P_t 2^f_t ( [s (c - 8)]_td + [b + 8 s]_tg )
// are one f16 operand each for keys and values, and the least values ride
// along as a few more columns, in two f16 parts: 32 more slots of the first
// product's depth (Q_g in two parts against them), one more tile of 16 columns
// of the second.  2^f_t joins the exponent, so the numerators that f16 has to
// hold are at most 2^15 whatever the steps of a row's tokens are.  What is left
// for a wave and (row, token) is the softmax: two products, a maximum, an
// exponential, a sum and the conversion.
//
// One step is 64 tokens of 128 dims or 32 of 256 (32 KB of operands, in two
// buffers: two workgroups a compute unit).  The wave that converts codes of
// group g for the products loads them two steps ahead; the pairs (s, b) go a
// step before them, through a ring of three.
//
// Measured: 2048 f32 rows of 16 x 256 from an empty context 133 us and 21 to
// join their parts; 4 x 4096 bf16 rows of 32 x 128, ragged, 443 us, 0.63
// PFLOP/s of the mathematics' operations.  In the f32 form 432 vector and 66
// matrix instructions a step and wave, 2770 of the 4450 cycles that a SIMD has
// for one with two waves on it; the rest is the longest block's tail, a part
// of 17 tiles of 64 tokens starting where another ends.  Blocks of 128 rows
// hold two operands of rows a wave: bf16 at 128 dims has the registers.
#include <hip/hip_runtime.h>

#include "attnq4_many.h"
#include "kvq4_host.h"

namespace chk {

uint32_t attn_q4_block(uint32_t hd, uint32_t dtype) { return hd == 128 && dtype == CHK_BF16 ? 128u : 64u; }

void launch_attn_q4_many(const AttnQ4Args& a, uint32_t hd, uint32_t dtype, uint32_t grid, hipStream_t st) {
    if (hd == 128) {
        if (dtype == CHK_F32) kv4_launch(k_attn_q4_rows<128, float, 1, Q4_ALL>, dim3(grid), CHK_WG, st, a);
        else if (dtype == CHK_F16) kv4_launch(k_attn_q4_rows<128, _Float16, 1, Q4_ALL>, dim3(grid), CHK_WG, st, a);
        else kv4_launch(k_attn_q4_rows<128, __bf16, 2, Q4_ALL>, dim3(grid), CHK_WG, st, a);
    } else {
        if (dtype == CHK_F32) kv4_launch(k_attn_q4_rows<256, float, 1, Q4_ALL>, dim3(grid), CHK_WG, st, a);
        else if (dtype == CHK_F16) kv4_launch(k_attn_q4_rows<256, _Float16, 1, Q4_ALL>, dim3(grid), CHK_WG, st, a);
        else kv4_launch(k_attn_q4_rows<256, __bf16, 1, Q4_ALL>, dim3(grid), CHK_WG, st, a);
    }
}

}  // namespace chk
