// Launch interface between the kernels over the 8-bit cache (kv8.hip) and
// the torch-extension host code (kv8.cpp).
//
// How the cache lies in memory, for one layer and one of K / V:
//   codes  uint8  [B, kvH, nblk, 32 * hdp]   32 tokens are one block
//   scales fp32   [B, kvH, nblk]
//   tail   16 bit [B, kvH, 2, 32 * hdp]      raw values, slot = block & 1
// hdp is head_dim rounded up to one of FMA_KV8_WIDTHS. Inside a block the
// 32 * hdp values lie in the order in which the 64 lanes of a wave feed them
// to v_mfma_f32_16x16x32 (kidx / vidx in kv8.hip), which is possible because
// a block is written at once, when its last token arrives: every load of the
// attention kernel is 16 contiguous bytes a lane and needs no transpose.
#pragma once

#include <hip/hip_runtime.h>

#define FMA_KV8_BLOCK 32

// One layer of a cache. Pointers are to K; V lies *_v elements behind.
struct FmaKv8Layer {
  unsigned char* codes;
  float* scales;
  void* tail;
  long long codes_v, scales_v, tail_v;
  int batch, kv_heads, nblk, max_seq, hd, hdp;
  int fp8;   // else int8 (held biased by 128)
  int bf16;  // type of tail, keys, values and queries; else fp16
};

// Where each sequence's first new token lies and how many are its own:
// start / counts from the device where the pointer is set, else the number.
struct FmaKv8Span {
  const int* start;
  const int* counts;
  int start_i;
  int T;
  int held;  // tokens stored of every sequence, if not only those of the span
};

// Rows of a [B, T, H, hd] tensor with a contiguous last dimension.
struct FmaRows {
  const void* p;
  long long sb, st, sh;  // strides in elements
  int vec;               // rows start on 16-byte borders and hd % 8 == 0
};

struct FmaRope {
  const float* cos;
  const float* sin;
  int half;      // rotated pairs
  int table;     // rows of cos / sin; 0 = no rotation
  int pairs;     // (2i, 2i+1), else (i, i + half)
  float eps;
  const void* qw;
  const void* kw;
  int tab_vec;   // rows of the tables start on 16-byte borders
  int w_vec;     // the gains too, and hd % 8 == 0
};

// position of token (b, t): base + b * sb + t * st of an int32 / int64
// tensor, or start + t
struct FmaPos {
  const int* p32;
  const long long* p64;
  long long sb, st, start;
  int per_token;
};

// type: 0 bf16, 1 fp16, 2 fp32
extern "C" hipError_t fma_launch_qk_norm_rope(
    FmaRows q, FmaRows k, void* qo, void* ko, int B, int T, int q_heads,
    int kv_heads, int hd, int type, FmaRope rope, FmaPos pos,
    hipStream_t stream);

// q.p == nullptr: store only
extern "C" hipError_t fma_launch_kv8_append(FmaKv8Layer c, FmaKv8Span span,
                                            FmaRows q, FmaRows k, FmaRows v,
                                            void* qo, int q_heads,
                                            FmaRope rope, hipStream_t stream);

extern "C" hipError_t fma_launch_kv8_read(FmaKv8Layer c, const int* start,
                                          int start_i, const int* length,
                                          int length_i, int n, void* ko,
                                          void* vo, hipStream_t stream);

// How a call is spread: rows of one kv head that a workgroup takes, and parts
// that the blocks of a sequence are split into.
struct FmaKv8Plan {
  int tile, splits;
};
// max_len: tokens that a sequence may have
extern "C" FmaKv8Plan fma_kv8_attn_plan(const FmaKv8Layer* c, int T,
                                        int q_heads, int max_len, int cus);
// partials: fp32, rows * splits * (hdp + 2) of them where splits > 1
extern "C" hipError_t fma_launch_kv8_attention(FmaKv8Layer c, FmaKv8Span span,
                                               FmaRows q, void* out,
                                               int q_heads, float scale,
                                               float* partials,
                                               FmaKv8Plan plan,
                                               hipStream_t stream);
