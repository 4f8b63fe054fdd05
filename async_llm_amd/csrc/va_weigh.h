// Plans for attention weights: which query rows look at which tokens, by token.
//
// Attention walks a query row's tokens; weights want the sum over a token's rows.  So a plan turns the sub-request tables round:
// runs of pages that the same sub-requests read at the same places ("spans") each get the packed list of those sub-requests'
// rows, and a work item is a chunk of a span's tokens with a range of that list.  Every token that somebody sees lies in one
// span, so its keys are read once however many rows look at it, and one workgroup a kv head owns its sum.  The others lie in
// none: tokens between single slots of a page that nobody sees split its span.
#pragma once
#include <stdint.h>

#define VA_WEIGH_MAGIC 0x56415731  // "VAW1"
#define VA_WEIGH_HEADER_WORDS 24
#define VA_WEIGH_ITEM_WORDS 8
#define VA_WEIGH_JOIN_WORDS 8

// Spans whose tokens have more than one tile of 16 (row, q head) pairs are cut into tile items of this many tokens (16-bit rows and
// codes, head dims of the matrix cores), the others into items of strips: see va_weigh.hip.
#define VA_WEIGH_TILE_TOKENS 256
#define VA_WEIGH_TILE_ROWS 32  // (row, q head) pairs of a tile of tile items; 16 in strips

// header word indices
enum {
  VA_WH_MAGIC = 0,
  VA_WH_N_ITEMS,   // tile items first, then those of strips
  VA_WH_N_ROWS,    // packed rows, padded to whole tiles of (row, q head) pairs
  VA_WH_N_JOINS,
  VA_WH_N_PARTIALS,  // partial sums, in tokens (per kv head)
  VA_WH_N_PAGES,
  VA_WH_OFF_ITEMS,
  VA_WH_OFF_JOINS,
  VA_WH_OFF_PAGES,
  VA_WH_OFF_ROWS,  // three arrays of n_rows: sub-row (-1: padding), first token and end of what it sees of its span
  VA_WH_HQ,        // what the plan was made for
  VA_WH_HKV,
  VA_WH_D,
  VA_WH_PAGE,
  VA_WH_DTYPE,
  VA_WH_CODES,
  VA_WH_POOL_PAGES,
  VA_WH_N_SUBROWS,
  VA_WH_N_TILE_ITEMS,  // a multiple of 8, padding included
  VA_WH_N_TILE_ROWS,   // packed rows of spans in tile items: the first ones
  VA_WH_N_STRIPS,      // a multiple of 8
  VA_WH_OFF_STRIPS,  // [n_strips + 1]: strip s is the items [strips[s], strips[s + 1])
};

// item word indices (n_tok = 0: padding)
enum {
  VA_WI_PAGES = 0,   // first entry of the span's pages
  VA_WI_FIRST,       // first token of the chunk, within the span
  VA_WI_N_TOK,
  VA_WI_TILE_BEGIN,  // tiles of (row, q head) pairs
  VA_WI_TILE_END,
  VA_WI_PARTIAL,     // where its sums go, in tokens; -1: it adds them to the weights itself
};

// join word indices: chunks whose rows are split among items
enum {
  VA_WJ_PAGES = 0,
  VA_WJ_FIRST,
  VA_WJ_N_TOK,
  VA_WJ_PARTIAL,   // first of n_parts runs of n_tok partial sums
  VA_WJ_N_PARTS,
};
