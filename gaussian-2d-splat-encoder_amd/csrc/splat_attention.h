// C-ABI description of a cross attention (mirrors include/splat_render.h).
#pragma once

extern "C" {
typedef struct splat_attention {
  int dtype, B, H, Hk, D;                          // element type; images; query heads; key heads; values per head
  float scale;                                     // of the scores
  long long Lq, Lk;                                // queries and keys of an image
  long long qb, ql, qh, kb, kl, kh, vb, vl, vh;    // elements from image to image, token to token, head to head
  long long gb, gl, gh;                            // the same of the output's gradient (backward)
  long long mb, ml;                                // key_mask: bytes from image to image and from key to key
  const int* kv_lengths;                           // [B] keys of each image that count, the first ones; or NULL
  const unsigned char* key_mask;                   // [B, Lk], 0: the key is left out; or NULL
  void* rest;                                      // what the backward takes besides lse; or NULL: bfloat16: what the
                                                   // outputs' rounding left, like them; float32: inverse sums, like lse
} splat_attention;
}
