// C-ABI descriptions of the token operators (mirror include/splat_render.h).
#pragma once

extern "C" {
typedef struct splat_rotation {
  int axes, interleaved;         // axes (0: nothing turns, 4 at most); pairs of neighbours instead of halves of an axis' values
  int dims[4];                   // values of a head that each axis turns, even, at most 128 together
  double quarters[64];           // quarter turns of each pair per unit of its axis' position
} splat_rotation;

typedef struct splat_positions {
  const void* p;                 // NULL: none
  int type;                      // 0 float32, 1 int32, 2 int64
  long long pb, pl, pa;          // elements from image to image, token to token, axis to axis
} splat_positions;

typedef struct splat_cache {
  int dtype, B, Hk, D;           // element type; sequences; key heads; values per head
  int page, width;               // tokens of a page; pages of a sequence's table
  long long pages;               // pages of the cache
  void *k, *v;                   // [pages, page, Hk, D]
  unsigned char* live;           // [pages, page], 0: the token is left out; or NULL
  long long kp, kt, kh, vp, vt, vh, lp, lt;   // elements from page to page, token to token, head to head
  const int* tables;             // [B, width] pages of each sequence in order
  long long tb;                  // elements from table to table
  const int *lengths, *counts;   // [B] tokens of each sequence, the new ones among them; new tokens, or NULL for all T
} splat_cache;

typedef struct splat_token_norm {
  int dtype, C;                  // element type; channels
  long long M;                   // tokens
  int layer, post, next;         // layer norms instead of root-mean-square ones; the block's output is normed; y is
  int gate, act;                 // 0 none, 1 a float row for each of `segs` runs of tokens, 2 a row for each token; activation
  long long segs;                // rows of a gate of kind 1
  float eps, scale;
  long long xl, hl, gl, dyl, dnl;   // elements from token to token of x, h, the gate (kind 2), the gradients of y and n
} splat_token_norm;
}
