// Arguments of the decoding kernels (kv_cache.cu, decode_attn.cu, sample.cu), filled by the torch-facing
// checks (decode_host.cpp).
#pragma once

#include <vector_types.h>

#include <cstdint>

namespace hb {

// How a cache keeps its values: 16 bits as they are, or 8-bit codes with one exponent byte per head of a token (act8.cuh).
enum KvType : int { kKvBf16 = 0, kKvF16 = 1, kKvCodes = 2 };

// A paged cache: element (page, head, slot, d) of K is k[page * kp + head * kh + slot * ks + d], its exponent byte
// ke[page * kep + head * keh + slot].
struct KvPool {
  void *k, *v;
  uint8_t *ke, *ve;                // null unless type is kKvCodes
  long kp, kh, ks, vp, vh, vs;     // strides in elements
  long kep, keh, vep, veh;
  int pages, heads, size, dim;     // size: slots of a page
  uint32_t per_head, per_slot;     // 2^32 over heads and size, rounded down (below 2^32)
  int type;                        // KvType
};

// K and V of new tokens.
struct KvTokens {
  const void *k, *v;               // [n, heads, dim]
  long kt, kh, vt, vh;             // strides of a token and a head, in elements
  const int64_t* slots;            // [n]: page * size + slot; negative: no slot
  int n;
  bool f16;
  bool vec;                        // every row starts on a 16-byte boundary
};

struct DecodeArgs {
  KvPool pool;
  const void* q;                   // [seqs, heads_q, dim], the new tokens' queries
  long qt, qh;                     // strides in elements
  bool q_vec;                      // query rows start on 16-byte boundaries
  bool f16;                        // of q and out
  const int* table;                // [seqs, width], row stride tt
  long tt;
  const int* lengths;              // [seqs]
  int longest;                     // tokens that a row of the table holds
  int seqs, heads_q;
  float scale;
  void* out;                       // [seqs, heads_q, dim]
  float* lse;                      // [seqs, heads_q]
  float* part;                     // per CTA, two unfinished units: maxima, sums and outputs of their columns
  int2* record;                    // and which they are: (unit or -1, CTAs behind that have more of it); null: CTAs take whole units
  int* status;
};

// How decode_attention deals out its work: a launch of `ctas` CTAs for each `seqs` sequences (0: more tiles than 32 bits
// count); `split`: a unit may be spread over CTAs.
struct DecodePlan {
  int seqs = 0, ctas = 0;
  bool split = false;
};

struct SampleArgs {
  const void* x;                   // [rows, >= V], row stride ld elements
  long ld;
  int type;                        // 0 bf16, 1 fp16, 2 fp32
  int rows, V;
  const float* u;                  // [rows]
  // each setting: one value per row, or (null) one for all
  const float* temperature;
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  double temperature0, top_p0, min_p0;
  int64_t top_k0;
  int64_t* tokens;                 // [rows]
};

}  // namespace hb
