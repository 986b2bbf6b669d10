// Addresses inside a tile of the paged 4-bit cache (16 tokens of one KV head), shared by the kernels that write it and
// those that read it.
//
// Codes are Q4_0's (value = d (code - 8), 32 dims per FP16 d). A 32-dim block is four 4-byte words; word w holds in byte i
// element 4 w + i (low nibble) and 16 + 4 w + i (high nibble), as bytes 4 w .. 4 w + 3 of a GGUF block do. The dims are
// cut into planes of four blocks (the last plane: what is left). Within a plane
//   K words lie [token][w][block]: lane (g, t) of a warp that takes token g's words w = t reads 16 bytes, the warp 512 in
//     a row, and holds for every block two k-steps of a 16 x 8 x 16 matrix instruction's B operand (dims along k);
//   V words lie [token / 8][token % 2][w][token / 2 % 4][block]: lane (g, t) that needs word w = g % 4 of the tokens
//     2 t + i (tokens along k) reads 16 bytes, again without bank conflicts.
// Behind the codes: K's scales, then V's, [token][block].
#pragma once
#include <cstdint>

namespace b200q {

__host__ __device__ inline unsigned kv4_plane_blocks(unsigned nb, unsigned p) {
    const unsigned left = nb - 4 * p;
    return left < 4 ? left : 4;
}
// byte offset in the tile of word w of block b, token t
__host__ __device__ inline unsigned kv4_k_word(unsigned nb, unsigned t, unsigned b, unsigned w) {
    const unsigned p = b / 4, n = kv4_plane_blocks(nb, p);
    return p * 1024 + ((t * 4 + w) * n + b % 4) * 4;
}
__host__ __device__ inline unsigned kv4_v_word(unsigned nb, unsigned t, unsigned b, unsigned w) {
    const unsigned p = b / 4, n = kv4_plane_blocks(nb, p);
    return nb * 256 + p * 1024 + ((((t / 8 * 2 + t % 2) * 4 + w) * 4 + t / 2 % 4) * n + b % 4) * 4;
}
__host__ __device__ inline unsigned kv4_k_scale(unsigned nb, unsigned t, unsigned b) { return nb * 512 + (t * nb + b) * 2; }
__host__ __device__ inline unsigned kv4_v_scale(unsigned nb, unsigned t, unsigned b) { return nb * 544 + (t * nb + b) * 2; }

}  // namespace b200q
