// What the kernels of attention over a shared prefix share (prefix_attn.cu, prefix_group.cu, prefix_latent.cu, and the forms of
// group_attn.cu / latent_attn.cu that finish it).
//
// Row r's keys are divided at own[r], a multiple of the page size: the positions below it lie in pages that several requests' page
// tables begin with, and are read once for all of them; the row reads the others by itself.  Softmax over a divided set of keys
// needs of every part only its maximum m, its sum l = sum exp(s - m) and its unnormalised result o = sum exp(s - m) v: with
// M = max m_i the whole is sum exp(m_i - M) o_i / sum exp(m_i - M) l_i.
//
// The plan is made on the host from the page tables (ops/prefix.py).  An item is a range of keys of one prefix and some of the
// rows that share it; the parts of row r are the cells cell[r] .. cell[r] + parts[r] - 1 of [cell][head].
#pragma once
#include <type_traits>

#include "ds41_stack.cuh"

namespace ds41 {

struct PrefixItem {
  int slot, first, rows, key0, key1, split;      // rows order[first] .. of the pass; keys [key0, key1) of the slot's page table
};
constexpr int kItemInts = 8;

__device__ __forceinline__ PrefixItem prefix_item(const ds41_prefix_plan& p, int i) {
  const int4 a = *reinterpret_cast<const int4*>(p.items + 1ll * i * kItemInts);
  const int2 b = *reinterpret_cast<const int2*>(p.items + 1ll * i * kItemInts + 4);
  return {a.x, a.y, a.z, a.w, b.x, b.y};
}

// a launch without a prefix
struct NoPrefix {};
template <typename X>
constexpr bool kHasPrefix = !std::is_same<X, NoPrefix>::value;

// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}

inline bool prefix_plan_ok(const ds41_prefix_plan* p) {
  return p != nullptr && p->items != nullptr && p->n_items != nullptr && p->order != nullptr && p->own != nullptr &&
         p->cell != nullptr && p->parts != nullptr && p->part_o != nullptr && p->part_ml != nullptr && p->max_items > 0 &&
         p->rows_per_item > 0 && p->grid > 0 && !(reinterpret_cast<uintptr_t>(p->items) & 15) &&
         !(reinterpret_cast<uintptr_t>(p->part_o) & 15) && !(reinterpret_cast<uintptr_t>(p->part_ml) & 7);
}

}  // namespace ds41
