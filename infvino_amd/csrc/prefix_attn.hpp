// Attention over a paged cache whose first pages the sequences of a group share, on gfx950 MFMA.
//
//   o[i] = (e^(m1 - m) o1 + e^(m2 - m) o2) / (e^(m1 - m) l1 + e^(m2 - m) l2),  m = max(m1, m2)
//
// with (m1, l1, o1) the maximum, sum and weighted values over the group's shared keys and (m2, l2, o2) those over
// the sequence's own: the shared keys are read once for the rows of all sequences, which are contiguous.
// Three kernels: shared keys, own keys, and the join of all parts.
#pragma once

#include "paged_attn.hpp"

namespace ivh {

namespace {

template <int TYPE> void launch_prefix_type(const PrefixParams & p, hipStream_t s)
{
  if (p.own.lead > 0) {
    if (p.own.c.bits == 8) launch_paged_dim<TYPE, 8, kSharedKeys>(p.first, s);
    else launch_paged_dim<TYPE, 16, kSharedKeys>(p.first, s);
  }
  if (p.own.c.bits == 8) launch_paged_dim<TYPE, 8, kOwnKeys>(p.own, s);
  else launch_paged_dim<TYPE, 16, kOwnKeys>(p.own, s);
  PagedParams join = p.own;
  join.parts = p.own.all_parts;
  launch_paged_join<TYPE>(join, s);
}

}  // namespace

}  // namespace ivh
