// f3s_kv4.cuh -- the 4-bit K/V page format, shared by the kernels that fill
// it (f3s_kv4_store.cu) and the attention that reads it (f3s_kv4_attend.cu).
//
// A page holds 16 tokens (the 16 rows of one block column).  Its record for
// one K/V head is 16 * D + 128 bytes:
//
//   K codes, 8 * D bytes: token-major rows of D / 2 bytes.  A 32-bit word
//     holds 8 consecutive channels c = 8 w + 2 n + h as the nibble n of its
//     16-bit half h.
//   V codes, 8 * D bytes: 16-bit halves, [p 2][g 8][t 4][w D/32][l 2]; the half
//     belongs to token 8 p + 2 t + l and its nibble n to channel
//     g * D / 8 + 4 w + n.
//   scales, 128 bytes: fp16 (scale, zero) of K and of V per token,
//     [token % 8][token / 8][K, V][scale, zero].
//
// A value is scale * (code - zero).  The order is that of the operands of
// mma.m16n8k16 with the cache as the 16-row A operand, so a lane's 8- or
// 16-byte load is its fragments:  for S^T = K Q^T the A rows are tokens and
// lane (g, t) = (lane / 4, lane % 4) holds channels t * D / 4 ... of tokens g
// and g + 8;  for O^T = V^T P^T the A rows are channels and the lane holds
// channels g * D / 8 ... of tokens 2t, 2t + 1, 2t + 8, 2t + 9.  No 16-bit half
// holds two tokens, so a token is stored with plain stores, without reading
// what its neighbours have there.
//
// A nibble becomes an fp16 number with one AND: nibble 0 (bits 0-3 of a
// half) is the subnormal code * 2^-24, nibble 1 (bits 4-7) code * 2^-20, and
// nibbles 2 and 3 the same after a shift by 8.  Both are exact, and the tensor
// cores multiply subnormals exactly; the two units are folded into Q (K's
// channels) and into the accumulators' rows (V's channels).
#pragma once
#include <cstdint>

namespace f3s {

constexpr int kPageTokens = 16;

__host__ __device__ constexpr int kv4_record_bytes(int d) { return 16 * d + 128; }

// byte offsets within a record
__host__ __device__ constexpr int kv4_k_off(int d, int token, int chunk8) { return token * (d / 2) + chunk8 * 4; }
__host__ __device__ constexpr int kv4_v_off(int d, int token, int g, int w) {
    return 8 * d + (token >> 3) * 4 * d + (g * 4 + ((token & 7) >> 1)) * (d / 8) + w * 4 + (token & 1) * 2;
}
__host__ __device__ constexpr int kv4_scale_off(int d, int token) {
    return 16 * d + (token & 7) * 16 + (token >> 3) * 8;
}

constexpr uint32_t kNib0 = 0x000f000fu;  // code * 2^-24
constexpr uint32_t kNib1 = 0x00f000f0u;  // code * 2^-20

// the smallest scale a row gets (a row of zeros): fp16's smallest number
constexpr float kKv4MinScale = 5.9604644775390625e-8f;
constexpr float kKv4MaxScale = 65504.f;

}  // namespace f3s
