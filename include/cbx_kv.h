/*
 * cbx_kv.h -- paged key/value caches of many streams on one MI355X: page
 * tables and slot maps built on the device from the streams' lengths, and
 * attention over the pages, a prompt that many streams share read once for
 * all of them.
 *
 * The reference holds one sequence's cache (src/main.cpp:419-424) and attends
 * over it (main.cpp:542-548).  cbx_t3.h's dense cache gives every stream n_ctx
 * positions; here a stream holds pages of page_size positions, as many as its
 * length needs, from a common pool, and streams of one voice share the pages
 * of that voice's prompt (speaker and conditioning rows, main.cpp:587-614).
 *
 * A serving loop: cbx_kv_build plans a call's rows (pages taken, where each
 * row's key and value go), then for every layer cbx_kv_attend stores them and
 * attends; cbx_t3_kv (cbx_t3.h) runs the whole transformer on such rows.
 *
 * Device pointers throughout, but for the structures themselves; every call
 * is asynchronous on `stream`, allocates nothing and holds nothing in the
 * handle, so it may be captured into a graph, and calls on buffers of their
 * own may run at once.
 */
#ifndef CBX_KV_H
#define CBX_KV_H

#include <stdint.h>

#include "cbx_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CBX_KV_F32 0 /* keys and values as computed                                  */
#define CBX_KV_F16 1 /* rounded to fp16 as they are stored (sums stay fp32)          */

/* The pool of pages: k[layer][page][head][position][64], v the same.  Heads
 * have 64 dimensions; n_head is the number of key/value heads. */
typedef struct cbx_kv_cache {
    void*   k;
    void*   v;
    int32_t type;       /* CBX_KV_*                                                  */
    int32_t n_layer;    /* >= 1                                                      */
    int32_t n_pages;    /* n_pages * page_size below 2^31                            */
    int32_t n_head;     /* >= 1                                                      */
    int32_t page_size;  /* 16, 32, 64, 128 or 256 positions                          */
} cbx_kv_cache;

/* Streams of the pool.  Streams [0, n_prefix) are prefixes: filled like any
 * other, then shared.  A stream i >= n_prefix whose parent[i] is one of them
 * sees that prefix's first prefix_len[i] positions (any number that calls
 * before have stored, also one that ends inside a page) as its own positions
 * [0, prefix_len[i]); its own pages begin there.  A prefix stays, and is not
 * released, as long as a stream shares it. */
typedef struct cbx_kv_streams {
    int32_t  n_streams;        /* 1 .. 16384                                         */
    int32_t  n_prefix;         /* 0 .. n_streams                                     */
    int32_t  max_pages;        /* pages a stream holds at most; max_pages * page_size
                                  below 2^30.  The step form's attention cuts rows
                                  by this capacity, not by their lengths: where it is
                                  many times the rows' it costs time                 */
    int32_t  n_pages;          /* the pool's                                         */
    int32_t* tables;           /* [n_streams][max_pages] page ids, in position order */
    int32_t* len;              /* [n_streams] positions stored in its own pages      */
    int32_t* free_pages;       /* [n_pages] a stack: entries [0, *n_free) are free   */
    int32_t* n_free;           /* [1]                                                */
    const int32_t* parent;     /* optional [n_streams]: a prefix, or -1              */
    const int32_t* prefix_len; /* [n_streams], required with parent                  */
} cbx_kv_streams;

/* The rows of one call, written by cbx_kv_build and read by the calls that
 * run on them.
 * Step form (stream NULL): row r is stream r's, n_rows = n_streams, one new
 * position a stream at most.
 * Prompt form (stream given): the streams' new positions one after the other,
 * in stream order; rows past the last have stream, position and slot -1. */
typedef struct cbx_kv_rows {
    int32_t  n_rows;
    int32_t  n_tiles;    /* entries of tiles: at least n_rows / tile_rows + n_streams
                            (prompt form) or + n_prefix (step form)                  */
    int32_t  tile_rows;  /* rows of a tile: cbx_kv_tile_rows(n_head, kv heads), 64
                            at most                                                  */
    int32_t* stream;     /* [n_rows] or NULL                                         */
    int32_t* position;   /* [n_rows], a prefix's positions counted; -1: no row       */
    int32_t* slot;       /* [n_rows] page * page_size + place in the page; -1: none  */
    int32_t* row_start;  /* [n_streams + 1] new rows before each stream              */
    int32_t* page_start; /* [n_streams + 1] pages taken before each stream           */
    int32_t* counts;     /* [4] rows, tiles, pages taken, streams refused            */
    int32_t* tiles;      /* [n_tiles][4] stream, first row, rows, keys.  Prompt form:
                            tile_rows rows of one stream, keys [0, keys); NULL with
                            n_tiles 0: the attention finds them from row_start.
                            Step form (optional): rows that share the prefix
                            `stream`, entries [first, first + rows) of order, keys
                            the longest of their prefixes.  Unused: -1, 0, 0, 0      */
    int32_t* order;      /* step form with tiles: [n_rows] the rows that share a
                            prefix, by prefix, then -1                               */
} cbx_kv_rows;

/* Rows of a tile for n_head query heads on n_kv_head key heads (at least 1,
 * n_head a multiple of n_kv_head): 64 (row, head) pairs of one key head, or one
 * row's where they are more. */
int32_t cbx_kv_tile_rows(int32_t n_head, int32_t n_kv_head);

/* One call's plan.  In this order, on the device: streams with release != 0
 * give their own pages back (to the top of the stack, in stream order) and have
 * length 0; every running stream asks for n_new positions (step form: for one
 * where n_new is not 0); pages are taken from the top of the stack in stream
 * order.  A stream is refused, and takes nothing, where its length would pass
 * max_pages * page_size (or is not in that range to begin with), where the rows
 * asked up to and with its own pass n_rows, or where it needs pages and those
 * needed up to and with its own are more than there are free.  counts tells
 * how many; a refused stream has no rows (row_start).
 * len and n_free become the new lengths and free count, or with len_out and
 * n_free_out those do and len and n_free are only read (both or neither). */
typedef struct cbx_kv_plan {
    const cbx_kv_streams* streams;
    const cbx_kv_rows*    rows;
    int32_t               page_size;
    const int32_t*        n_new;      /* optional [n_streams]; NULL: 1 each          */
    const int32_t*        state;      /* optional [n_streams]: only streams in
                                         CBX_DECODE_RUNNING ask                      */
    const int32_t*        release;    /* optional [n_streams]                        */
    int32_t*              len_out;    /* optional [n_streams]                        */
    int32_t*              n_free_out; /* [1] with len_out                            */
} cbx_kv_plan;

/* Page tables, rows and tiles of a call from the streams' lengths.  No
 * counterpart in the reference, whose one sequence fills one dense cache. */
int cbx_kv_build(cbx_sampler* s, const cbx_kv_plan* p, void* stream);

/* Attention of a layer's rows: out[r] = softmax(scale q[r] K^T) V over
 * positions [0, position[r]] of row r's stream, for each of n_head query heads
 * (head h reads key head h / (n_head / cache->n_head)).  With k and v, row r's
 * are first stored at slot[r] (rows of one stream in one call see each other's);
 * without, the cache holds them already.  Rows without a position give zeros;
 * a row with a position whose page is not one of the pool's does not see those
 * positions; a row that sees none gives zeros.  Keys and values that a row does
 * not see never reach it, whatever they hold.  A query or a seen key that is
 * not finite leaves its own row's outputs undefined, no other's; so does a score
 * of 2^127 or more, or a seen value of 2^80.
 * Sums and softmax statistics are fp32.  Products are fp32's, or on the 16-bit
 * matrix cores of values cut into parts: fp32 caches' into three bf16 parts
 * (each product to 2^-21 of itself, of values that are 0 or 2^-100 and more in
 * magnitude); fp16 caches' queries and weights into two
 * fp16 parts (to 2^-22 and 2^-20 of themselves, or 2^-38 of the row's largest).
 * n_rows * n_head, with tiles + n_tiles * cache->n_head (prompts without a list:
 * as many as it would have), is at most 2^24 - 1,
 * and n_pages * page_size * cache->n_head below 2^32 - 1 (CBX_ERR_UNSUPPORTED).
 * Step form with tiles: prefixes are read once for the rows of a tile; without:
 * by every row for itself, with the same result up to rounding. */
typedef struct cbx_kv_attn {
    const cbx_kv_cache*   cache;
    const cbx_kv_streams* streams;
    const cbx_kv_rows*    rows;
    int32_t      layer;
    int32_t      n_head;          /* query heads: a multiple of cache->n_head, at most
                                     64 times as many                                */
    const float* q;               /* [n_rows][ld_q], head h at 64 h                  */
    int64_t      ld_q;            /* >= 64 n_head, a multiple of 4                   */
    const float* k;               /* optional [n_rows][ld_kv], key head h at 64 h    */
    const float* v;               /* with k                                          */
    int64_t      ld_kv;           /* >= 64 cache->n_head, a multiple of 4, < 2^31    */
    float*       out;             /* [n_rows][ld_out], apart from q, k and v         */
    int64_t      ld_out;          /* >= 64 n_head, a multiple of 4                   */
    float        scale;
    void*        workspace;       /* cbx_kv_workspace_bytes of this call; 16-byte
                                     aligned, as q, k, v, out and the caches         */
    uint64_t     workspace_bytes;
} cbx_kv_attn;

/* Bytes of workspace a call needs (0: none; also 0 where the sizes are not
 * ones that cbx_kv_attend takes). */
uint64_t cbx_kv_workspace_bytes(const cbx_kv_attn* a);

/* Replaces main.cpp:542-548 (and the stores of :517-531) of one layer for many
 * streams. */
int cbx_kv_attend(cbx_sampler* s, const cbx_kv_attn* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
