// Launchers behind mtj_k_cache_attn: few new tokens (mtj_cache_few.cu) and prompts (mtj_cache_prompt.cu).
#pragma once
#include "mtj_cache.cuh"
#include "mtj_kernels.h"

namespace mtj {

constexpr int kFewBatch = 256;             // sequences of a launch; larger batches take several

struct CacheFewArgs {
  mtj_cache_attn_args c;                   // pointers from the launch's first sequence on
  int t0, tokens;                          // the launch's tokens of the call's
  float scale_log2;                        // score scale times log2(e)
  int score_rows;                          // rows of a key's scores
  int aligned, whole;                      // pieces end where units do; every unit is one piece
  int least, teams;                        // tiles of a piece at least, and the multiple that it is of
  int pieces;                              // blocks of the launch
  int32_t* prefix;                         // [kFewBatch + 1] tiles before each sequence
  int32_t* unit_blocks;                    // [units][2] the first and the last block that worked on a unit
  float2* part_ml;                         // [pieces][2][tile rows]: maximum (base 2), sum
  float* part_o;                           // [pieces][2][tile rows][d_head]
  float2* lse;                             // [units][tile rows] of units that one block had, with weights
  float* scores;                           // [tiles][keys][score_rows] (base 2), with weights
};
// Tile where piece k of the n of a unit begins, the unit's end for k = n: floor(tiles k / n).  The product itself leaves 32 bits in
// units of more than 2^31 / 296 tiles, 2^27 slots of 256-wide heads.
__host__ __device__ __forceinline__ int unit_piece_begin(int tiles, int n, int k) { return tiles / n * k + tiles % n * k / n; }
// How many blocks worked on a unit, from what its first and its last one wrote down; 0 where they did not both: a block whose wait ran out
// leaves out the rest of its piece, and the scratch holds anything there.
__host__ __device__ __forceinline__ int unit_blocks_of(int first, int last, int pieces) {
  return first >= 0 && first <= last && last < pieces ? last - first + 1 : 0;
}
struct CacheFewPlan {
  int tokens, batch, tile_rows, pieces, score_rows, aligned, whole, least, teams;
  int64_t prefix_off, units_off, ml_off, o_off, lse_off, scores_off, total;
};
CacheFewPlan plan_cache_few(const mtj_cache_attn_args& c);
cudaError_t run_cache_few(const mtj_cache_attn_args& c, const CacheFewPlan& p, char* scratch, cudaStream_t s);
// Prompts, bf16 without weights (mtj_cache_prompt.cu).
int64_t cache_prompt_scratch(const mtj_cache_attn_args& c);
bool cache_prompt_fits(const mtj_cache_attn_args& c);      // the new tokens of a sequence, into a launch's plan
cudaError_t run_cache_prompt(const mtj_cache_attn_args& c, char* scratch, cudaStream_t s);

// eight numbers of a row as bf16, rounded where they are not
__device__ __forceinline__ uint4 load8_bf16(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint4 load8_bf16(const float* p) {
  const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
  return make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}
// eight results times f
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v, float f) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0] * f, v[1] * f), pack_bf16x2(v[2] * f, v[3] * f),
                                            pack_bf16x2(v[4] * f, v[5] * f), pack_bf16x2(v[6] * f, v[7] * f));
}
__device__ __forceinline__ void store8(float* p, const float* v, float f) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
}

}  // namespace mtj
