// The paged K / V cache on the device: page geometry and the checks of a caller's rf_pages.
#pragma once
#include "rf_common.h"

namespace rf {

// rf_pages by value, with the page size as a shift and the strides of a head inside a page.
struct PagesDev {
  char* k;
  char* v;
  uint8_t* ks;
  uint8_t* vs;
  int64_t page_stride, scale_stride;   // bytes from a page to the next
  int64_t n_pages;
  int head_bytes, head_scales;         // bytes of one head of a page: values, scales
  int shift;                           // log2(tokens a page)
};

inline int log2_of(int p) {
  int s = 0;
  while ((1 << s) < p) ++s;
  return s;
}

// RF_OK and `d` filled, or a refusal naming fn.
inline int check_pages(const char* fn, const rf_pages* p, PagesDev* d) {
  if (!p || !p->k || !p->v) return fail(RF_EINVAL_ARG, "%s: null pointer (pages)", fn);
  if (p->kind != RF_PAGES_BF16 && p->kind != RF_PAGES_MX4) return fail(RF_EINVAL_ARG, "%s: kind of pages %d", fn, p->kind);
  if (p->d != 64 && p->d != 128 && p->d != 256)
    return fail(RF_EUNSUPPORTED, "%s: head_dim %d (the kernels take 64, 128, 256)", fn, p->d);
  if (p->page < 16 || p->page > 1024 || (p->page & (p->page - 1)))
    return fail(RF_EINVAL_SHAPE, "%s: %d tokens a page (a power of two from 16 to 1024)", fn, p->page);
  // (a head of a page is addressed with 32 bits, pages with 64)
  if (p->hkv <= 0 || p->hkv > 4096 || p->n_pages <= 0 || p->n_pages > INT32_MAX)
    return fail(RF_EINVAL_SHAPE, "%s: %lld pages of %d heads", fn, (long long)p->n_pages, p->hkv);
  const bool mx = p->kind == RF_PAGES_MX4;
  const int64_t head = static_cast<int64_t>(p->page) * p->d * (mx ? 1 : 4) / 2, scales = static_cast<int64_t>(p->page) * p->d / 32;
  if (p->page_stride < p->hkv * head || p->page_stride % 16 || !aligned16(p->k) || !aligned16(p->v))
    return fail(RF_EINVAL_SHAPE, "%s: page stride %lld bytes (at least %lld, a multiple of 16) or alignment", fn,
                (long long)p->page_stride, (long long)(p->hkv * head));
  if (mx) {
    if (!p->ks || !p->vs) return fail(RF_EINVAL_ARG, "%s: null pointer (scales)", fn);
    if (p->scale_stride < p->hkv * scales || p->scale_stride % 8 || (reinterpret_cast<uintptr_t>(p->ks) & 7u) ||
        (reinterpret_cast<uintptr_t>(p->vs) & 7u))
      return fail(RF_EINVAL_SHAPE, "%s: scale stride %lld bytes (at least %lld, a multiple of 8) or alignment", fn,
                  (long long)p->scale_stride, (long long)(p->hkv * scales));
  }
  *d = PagesDev{static_cast<char*>(p->k), static_cast<char*>(p->v), p->ks, p->vs, p->page_stride, p->scale_stride,
                p->n_pages, static_cast<int>(head), static_cast<int>(scales), log2_of(p->page)};
  return RF_OK;
}

typedef __bf16 rf_fp4_pair __attribute__((ext_vector_type(2)));

// The two bf16 values (low half: the byte's low code) of byte J of the codes in w, times a scale 2^n. Both codes and
// scale are exact in bf16; a scale whose exponent bits are all ones gives NaN.
template <int J>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, J));
}

// The scale that byte I of w stands for, 2^(byte - 127); 255 has the exponent bits of NaN.
template <int I>
__device__ __forceinline__ float scale_of(uint32_t w) {
  return __uint_as_float((I == 3 ? w >> 1 : w << (23 - 8 * I)) & 0x7f800000u);
}

}  // namespace rf
