// Argument checks that the entry points over packed rows and the paged cache share.
#pragma once

#include "common.hpp"

namespace tt {

inline int check_heads(const char* what, int tokens, int batch, int heads, int kv_heads, int head_dim, int dtype) {
  TT_REQUIRE(tokens >= 0 && batch >= 0, "%s: bad shape (tokens %d, batch %d)", what, tokens, batch);
  TT_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "%s: heads %d are no multiple of kv_heads %d", what,
             heads, kv_heads);
  TT_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0, "%s: head_dim %d is no multiple of 8 up to 256",
             what, head_dim);
  TT_REQUIRE((int64_t)tokens * heads < (1LL << 31), "%s: %d rows of %d heads", what, tokens, heads);
  TT_REQUIRE(dtype == TT_FP16 || dtype == TT_BF16, "%s: bad dtype %d", what, dtype);
  return TT_OK;
}

// Rows and heads are read 16 bytes at a time, and 16 rows at an offset of 32 bits.
inline int check_rows(const char* what, const void* p, int64_t row, int64_t head) {
  TT_REQUIRE(((uintptr_t)p & 15) == 0 && row % 8 == 0 && head % 8 == 0, "%s: not aligned to 16 bytes", what);
  TT_REQUIRE(row >= 0 && head >= 0 && row < (1LL << 26), "%s: row stride of %lld elements", what, (long long)row);
  return TT_OK;
}

inline int check_pages(const char* what, int pages, int page_size, int table_pages) {
  TT_REQUIRE(pages > 0 && table_pages > 0, "%s: no pages (%d in the cache, %d per sequence)", what, pages, table_pages);
  TT_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0, "%s: page_size %d is no power of two from 16 on",
             what, page_size);
  TT_REQUIRE((int64_t)page_size * table_pages <= (1LL << 30), "%s: %d pages of %d per sequence", what, table_pages,
             page_size);
  return TT_OK;
}

// A cache in 8 bits: rows and heads 16 bytes apart, a scale for each `block` tokens of a page and head.
inline int check_head8(const char* what, int head_dim) {
  TT_REQUIRE(head_dim % 16 == 0, "%s: head_dim %d is no multiple of 16, which a cache in 8 bits needs", what, head_dim);
  return TT_OK;
}

inline int check_rows8(const char* what, const void* p, int64_t page, int64_t row, int64_t head) {
  TT_REQUIRE(((uintptr_t)p & 15) == 0 && page % 16 == 0 && row % 16 == 0 && head % 16 == 0, "%s: not aligned to 16 bytes",
             what);
  TT_REQUIRE(page >= 0 && row >= 0 && head >= 0 && row < (1LL << 26), "%s: strides of %lld, %lld and %lld bytes", what,
             (long long)page, (long long)row, (long long)head);
  return TT_OK;
}

inline int check_block(const char* what, int block, int page_size) {
  TT_REQUIRE(block >= 16 && block <= page_size && block <= 65536 && (block & (block - 1)) == 0,
             "%s: a scale for each %d tokens of pages of %d (powers of two, from 16 to 65536)", what, block, page_size);
  return TT_OK;
}

// (After check_block: an offset into the scales has 32 bits.)
template <class C>
int check_scales(const char* what, const C& c) {
  TT_REQUIRE(c.k_scales != nullptr && c.v_scales != nullptr, "%s: null pointer", what);
  const int64_t most = 1LL << 31, blocks = c.page_size / c.block;
  TT_REQUIRE(c.s_page >= 0 && c.s_block >= 0 && c.s_head >= 0 && c.s_page < most && c.s_block < most && c.s_head < most &&
                 (c.pages - 1) * c.s_page < most && (blocks - 1) * c.s_block < most && (c.kv_heads - 1) * c.s_head < most &&
                 (c.pages - 1) * c.s_page + (blocks - 1) * c.s_block + (c.kv_heads - 1) * c.s_head < most,
             "%s: scales %lld, %lld and %lld bytes apart do not lie within 2 GiB", what, (long long)c.s_page,
             (long long)c.s_block, (long long)c.s_head);
  return TT_OK;
}

// What a call writes: `n` of them lie apart.
inline int check_apart(const char* what, const char* of, int64_t stride, int64_t n) {
  TT_REQUIRE(stride > 0 || n <= 1, "%s: %lld %s at one address", what, (long long)n, of);
  return TT_OK;
}

}  // namespace tt

#define TT_CHECK(call)            \
  do {                            \
    const int rc_ = (call);       \
    if (rc_ != TT_OK) return rc_; \
  } while (0)

// The structure is the caller's: its size first.
#define TT_ARGS(type, what)                                                                             \
  TT_REQUIRE(args != nullptr && args->size == (int64_t)sizeof(type), what ": not a " #type " structure"); \
  const type& c = *args
