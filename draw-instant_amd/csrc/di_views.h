// Host-side checks of the head views (di_heads) that the attention-layer
// entry points take: every element a view names lies in its buffer, and two
// views that are read and written by one call do not overlap.
#pragma once

#include <cstdint>

#include "di_internal.h"

namespace di {

// A checked view: element (b, s, h, c) at p[b * batch + s * token + h * head + c].
struct HeadsPtr {
  char* p;          // first element of the view
  uint64_t token, head, batch;  // strides in elements
  uint64_t buf;     // handle, first and one-past-last element: for overlap checks
  uint64_t first, end;
  uint64_t width;   // elements of one token's heads: (H - 1) * head + d
};

constexpr uint64_t kMaxStride = 1ull << 40;

inline int check_heads(Ctx* c, const di_heads* v, const char* fn, const char* name, uint64_t B, uint64_t S,
                       uint64_t H, uint64_t d, int dt, HeadsPtr* out) {
  DI_REQUIRE(v != nullptr, DI_EINVAL, "%s: null view %s", fn, name);
  DI_REQUIRE(v->offset < kMaxStride && v->token < kMaxStride && v->head < kMaxStride && v->batch < kMaxStride,
             DI_EINVAL, "%s: offset or stride of %s past 2^40 elements", fn, name);
  Buffer* b = nullptr;
  const int rc = lookup(c, v->buf, &b);
  if (rc) return rc;
  const size_t es = dtype_size(dt);
  // (strides below 2^40, counts below 2^32: the sum in 128 bits)
  const unsigned __int128 end = (unsigned __int128)v->offset + (unsigned __int128)(B - 1) * v->batch +
                                (unsigned __int128)(S - 1) * v->token + (unsigned __int128)(H - 1) * v->head + d;
  DI_REQUIRE(end * es <= b->bytes, DI_EINVAL, "%s: view %s ends past its buffer of %llu bytes", fn, name,
             (unsigned long long)b->bytes);
  out->p = (char*)b->ptr + v->offset * es;
  out->token = v->token;
  out->head = v->head;
  out->batch = v->batch;
  out->buf = v->buf;
  out->first = v->offset;
  out->end = (uint64_t)end;
  out->width = (H - 1) * v->head + d;
  return DI_OK;
}

// No two elements of a written view share a place: each of its dimensions
// (those of more than one entry, by stride) steps past all that lies below it.
inline bool heads_distinct(const HeadsPtr& v, uint64_t B, uint64_t S, uint64_t H, uint64_t d) {
  uint64_t st[3] = {v.token, v.head, v.batch}, n[3] = {S, H, B};
  for (int i = 0; i < 2; i++)
    for (int j = 0; j < 2 - i; j++)
      if (st[j] > st[j + 1]) {
        const uint64_t a = st[j], b = n[j];
        st[j] = st[j + 1], n[j] = n[j + 1];
        st[j + 1] = a, n[j + 1] = b;
      }
  unsigned __int128 extent = d;
  for (int i = 0; i < 3; i++) {
    if (n[i] <= 1) continue;
    if (st[i] < extent) return false;
    extent += (unsigned __int128)(n[i] - 1) * st[i];
  }
  return true;
}

// Whether a written view and another one touch a common element, as far as
// can be told without counting: apart in their buffer, or in columns of the
// same token rows that do not meet.  (Two that pass neither are taken to overlap.)
inline bool heads_apart(const HeadsPtr& a, const HeadsPtr& b) {
  if (a.buf != b.buf || a.end <= b.first || b.end <= a.first) return true;
  if (a.token == 0 || a.token != b.token || a.batch != b.batch || a.batch % a.token != 0) return false;
  const uint64_t ca = a.first % a.token, cb = b.first % a.token;
  if (ca + a.width > a.token || cb + b.width > a.token) return false;
  return ca + a.width <= cb || cb + b.width <= ca;
}

inline bool heads_same(const HeadsPtr& a, const HeadsPtr& b) {
  return a.buf == b.buf && a.first == b.first && a.token == b.token && a.head == b.head && a.batch == b.batch;
}

// Every row starts on a multiple of `n` elements.
inline bool heads_aligned(const HeadsPtr& v, uint64_t n) {
  return v.first % n == 0 && v.token % n == 0 && v.head % n == 0 && v.batch % n == 0;
}

}  // namespace di
