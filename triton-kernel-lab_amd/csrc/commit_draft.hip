// The accepted nodes' move into the KV cache: row seqlens[b] + i of every KV head takes row
// path[b][i] of the drafted tokens' keys and values, i < count[b]. One 16-byte chunk of a key
// and a value per thread, all (batch, head) pairs in one launch: the call moves at most a few MB,
// so what counts is one trip to memory for the path and one for the rows.
#include "tk_common.hpp"

namespace {

struct CommitArgs {
  char* cache[2];
  const char* tree[2];
  const int32_t* seqlens;
  const int32_t* path;
  const int32_t* count;
  int32_t* new_seqlens;
  int64_t cache_s[2][3], tree_s[2][3];  // bytes, {batch, head, position}
  int max_len, nodes, chunks;           // 16-byte chunks per row
};

// One 16-byte chunk of a row of K and V per thread.
__global__ __launch_bounds__(256) void commit_kernel(CommitArgs a) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int idx = blockIdx.x * 256 + threadIdx.x;
  const int len = min(max(a.seqlens[b], 0), a.max_len);
  const int count = min(max(a.count[b], 0), a.nodes);
  if (idx == 0 && h == 0) a.new_seqlens[b] = len + min(count, a.max_len - len);
  const int i = idx / a.chunks, c = idx - i * a.chunks;
  if (i >= count || len + i >= a.max_len) return;
  const int node = a.path[int64_t(b) * a.nodes + i];
  if (node < 0 || node >= a.nodes) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const char* src = a.tree[w] + b * a.tree_s[w][0] + h * a.tree_s[w][1] +
                      node * a.tree_s[w][2] + c * 16;
    char* dst = a.cache[w] + b * a.cache_s[w][0] + h * a.cache_s[w][1] +
                int64_t(len + i) * a.cache_s[w][2] + c * 16;
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  }
}

}  // namespace

extern "C" int tk_commit_draft(int dtype, void* k_cache, void* v_cache, const void* k_tree,
                               const void* v_tree, const int32_t* seqlens, const int32_t* path,
                               const int32_t* count, int32_t* new_seqlens, int64_t batch,
                               int64_t kv_heads, int64_t max_len, int64_t nodes,
                               int64_t head_dim, const int64_t* k_cache_strides,
                               const int64_t* v_cache_strides, const int64_t* k_tree_strides,
                               const int64_t* v_tree_strides, void* stream) {
  if (dtype != TK_DTYPE_F16 && dtype != TK_DTYPE_BF16)
    return tk::fail("commit draft: dtype must be float16 or bfloat16");
  if (k_cache == nullptr || v_cache == nullptr || k_tree == nullptr || v_tree == nullptr ||
      seqlens == nullptr || path == nullptr || count == nullptr || new_seqlens == nullptr ||
      k_cache_strides == nullptr || v_cache_strides == nullptr || k_tree_strides == nullptr ||
      v_tree_strides == nullptr)
    return tk::fail("commit draft: null pointer");
  if (batch <= 0 || kv_heads <= 0 || max_len <= 0 || nodes <= 0 || head_dim <= 0)
    return tk::fail("commit draft: empty problem");
  if (head_dim % 8 != 0) return tk::fail("commit draft: head_dim must be a multiple of 8");
  if (batch > 65535 || kv_heads > 65535 || max_len > INT32_MAX / 2 || nodes > 65535 ||
      head_dim > 65535)
    return tk::fail("commit draft: problem too large");
  CommitArgs a;
  a.cache[0] = static_cast<char*>(k_cache);
  a.cache[1] = static_cast<char*>(v_cache);
  a.tree[0] = static_cast<const char*>(k_tree);
  a.tree[1] = static_cast<const char*>(v_tree);
  const int64_t* cache_s[2] = {k_cache_strides, v_cache_strides};
  const int64_t* tree_s[2] = {k_tree_strides, v_tree_strides};
  for (int w = 0; w < 2; ++w) {
    if (!tk::aligned16(a.cache[w]) || !tk::aligned16(a.tree[w]))
      return tk::fail("commit draft: tensors must be 16-byte aligned");
    for (int d = 0; d < 3; ++d) {
      for (int64_t st : {cache_s[w][d], tree_s[w][d]})
        if (st < 0 || st % 8 != 0 || st >= (int64_t(1) << 40))
          return tk::fail("commit draft: strides must be non-negative multiples of 8 elements");
      a.cache_s[w][d] = cache_s[w][d] * 2;
      a.tree_s[w][d] = tree_s[w][d] * 2;
    }
  }
  a.seqlens = seqlens;
  a.path = path;
  a.count = count;
  a.new_seqlens = new_seqlens;
  a.max_len = static_cast<int>(max_len);
  a.nodes = static_cast<int>(nodes);
  a.chunks = static_cast<int>(head_dim / 8);
  const dim3 grid(static_cast<uint32_t>(tk::cdiv(nodes * a.chunks, 256)),
                  static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(batch));
  hipLaunchKernelGGL(commit_kernel, grid, dim3(256), 0, tk::as_stream(stream), a);
  return tk::check_launch("commit draft");
}
