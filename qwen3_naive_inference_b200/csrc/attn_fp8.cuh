// Host side shared by the attentions over the 8-bit paged KV cache: argument checks, tensor maps.
#pragma once
#include <atomic>

#include "kv_fp8.cuh"
#include "tma.cuh"

namespace {

constexpr float KV8_LOG2E = 1.4426950408889634f;
constexpr int KV8_MAX_GROUP = 16;  // query heads of a kv head

// Lets kernel `fn` have `bytes` of dynamic shared memory on the current device; `done` holds a bit per
// device that it was asked for on.
int kv8_allow_smem(const void* fn, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return qb_launch_status();
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return QB_OK;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return qb_launch_status();
  done.fetch_or(bit, std::memory_order_relaxed);
  return QB_OK;
}

int kv8_check_cache(const void* q, int64_t q_stride, const void* k, const void* v, const float* ks, const float* vs,
                    int64_t num_blocks, const int32_t* bt, int64_t bt_stride, int bt_width, int hq, int hkv,
                    const void* out) {
  const auto al16 = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  QB_CHECK_ARG(hq > 0 && hkv > 0 && hq % hkv == 0 && hq / hkv <= KV8_MAX_GROUP);
  QB_CHECK_ARG(al16(q) && al16(out) && al16(k) && al16(v) && ks && vs && bt);
  QB_CHECK_ARG(q_stride >= (int64_t)hq * KV8_D && q_stride % 8 == 0 && bt_stride >= 0 && bt_width >= 0);
  // rows of codes are counted in 32 bits (2^31 of them are 256 GB)
  QB_CHECK_ARG(num_blocks > 0 && num_blocks <= (int64_t)INT32_MAX / KV8_PAGE / hkv);
  return QB_OK;
}

// The cache as [num_blocks * hkv * 256, 128] bytes, read `rows` rows of a block of 64 at a time; the 16-byte
// chunks of a row are XORed with (row & 7), so that eight rows' chunks lie in different banks.
bool kv8_tmap(CUtensorMap* map, const void* codes, int64_t num_blocks, int hkv, int rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)KV8_D, (cuuint64_t)num_blocks * hkv * KV8_PAGE};
  cuuint64_t strides[1] = {(cuuint64_t)KV8_D};
  cuuint32_t box[2] = {(cuuint32_t)KV8_D, (cuuint32_t)rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
