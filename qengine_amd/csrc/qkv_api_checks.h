// qkv_api_checks.h -- argument checks shared by the files of the C ABI around the paged 8-bit
// cache (qkv_api_paged8.cpp, qkv_api_loop.cpp).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/qkv.h"
#include "qkv_launch.h"

namespace {

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
inline int launch_status(hipError_t e) { return e == hipSuccess ? QKV_OK : QKV_ERR_LAUNCH; }

// entries of a fork or release: a launch of 256 threads each drops what is past 2^32 threads
constexpr int kMaxList = 1 << 24;

constexpr qkv::PageStatus kPageStatus{QKV_OK, QKV_ERR_INVALID, QKV_ERR_PAGES};

// the shape of a paged 8-bit cache
inline int check_f8_pool(int num_kv, int head_dim, int max_blocks, int block_tokens, int n_pages) {
  if (head_dim != 128 && head_dim != 256) return QKV_ERR_UNSUPPORTED;
  if (num_kv <= 0 || max_blocks <= 0 || block_tokens <= 0 || n_pages <= 0) return QKV_ERR_INVALID;
  if (block_tokens % 16) return QKV_ERR_UNSUPPORTED;
  // (the kernels address inside a page in 32 bits)
  if ((double)block_tokens * num_kv * head_dim > 2147483647.0) return QKV_ERR_UNSUPPORTED;
  return QKV_OK;
}

inline int check_tables(const qkv::PageTables& t) {
  if (t.n_slots <= 0 || t.max_blocks <= 0 || t.block_tokens <= 0 || t.n_pages <= 0) return QKV_ERR_INVALID;
  if (!t.tables || !t.refs) return QKV_ERR_NULL;
  if (!aligned(t.tables, 4) || !aligned(t.refs, 4)) return QKV_ERR_ALIGN;
  return QKV_OK;
}

inline int take_planes(const qkv_page_plane* planes, int n, qkv::PagePlanes& out) {
  if (n < 0) return QKV_ERR_INVALID;
  if (n > qkv::kMaxPlanes) return QKV_ERR_UNSUPPORTED;
  if (n > 0 && !planes) return QKV_ERR_NULL;
  out.n = n;
  for (int i = 0; i < n; i++) {
    if (!planes[i].base) return QKV_ERR_NULL;
    if (planes[i].page_bytes == 0 || planes[i].page_bytes > 0x7fffffffULL) return QKV_ERR_INVALID;
    out.base[i] = static_cast<uint8_t*>(planes[i].base);
    out.bytes[i] = planes[i].page_bytes;
  }
  return QKV_OK;
}

}  // namespace
