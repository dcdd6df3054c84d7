// The merge kernel of prefix attention on records made by a test
// (test_gpu_attention_merge.py): what it makes of those that a test cannot
// have the other kernels write, such as the ones of a wait that ran out.
#include "../miniserve_b200/csrc/ms_attn.cuh"

extern "C" {

float record_bad_page() { return ms::kAtBadPage; }
float record_late() { return ms::kAtLate; }

// `splits` records of every query head, no own keys; bf16 heads of 64.
int merge_records(int wide, int rows, int heads, int kv_heads, int splits, const float *o, const float *ml,
                  const int32_t *lengths, int64_t *base, int64_t *header, void *out, float *lse, int32_t *status,
                  void *stream) {
  ms::AtArgs a{};
  a.x.rows = rows, a.x.heads = heads, a.x.kv_heads = kv_heads, a.x.head_dim = 64;
  a.x.lengths = lengths, a.x.page_size = 16;
  a.x.out = out, a.x.out_row = heads * 64, a.x.out_head = 64, a.x.lse = lse, a.x.status = status;
  a.shape.rows = rows, a.shape.heads = heads, a.shape.kv_heads = kv_heads, a.shape.head_dim = 64;
  a.shape.group = heads / kv_heads;
  a.shape.chunks = (a.shape.group + ms::kAtRows - 1) / ms::kAtRows;
  a.shape.chunk_rows = a.shape.group < ms::kAtRows ? a.shape.group : ms::kAtRows;
  a.header = reinterpret_cast<ms::AtHeader *>(header);
  a.base = base;
  a.packed = rows * a.shape.group;
  a.pre_splits = splits;
  a.pre_o = const_cast<float *>(o);
  a.pre_ml = reinterpret_cast<float2 *>(const_cast<float *>(ml));
  const int outputs = rows * heads;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide)
    ms::ms_attn_merge_kernel<__nv_bfloat16, 64, ms::kMgWide><<<outputs, ms::kMgWide * 32, 0, s>>>(a);
  else
    ms::ms_attn_merge_kernel<__nv_bfloat16, 64, 1>
        <<<(outputs + ms::kMgNarrow - 1) / ms::kMgNarrow, ms::kMgNarrow * 32, 0, s>>>(a);
  return (int)cudaGetLastError();
}
}
