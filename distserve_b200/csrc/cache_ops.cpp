// Operator shim of the cache's contents: torch.ops.kv_cache_ops.{write,read} and
// torch.ops.kv_attention_ops.{paged,prompt} over the C ABI of libkvmig.so.  Part of libst_pybinding.so.
//
// Like the other operators' shim it only unpacks tensors, makes their device current for the call, picks up that
// device's current stream and turns a status into an exception.
#include <torch/library.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../include/kvmig.h"

namespace {

void check(int64_t rc, const char* op) {
    TORCH_CHECK(rc >= 0, op, ": ", kvmig_last_error(), " (kvmig status ", rc, ")");
}

int dtype_of(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be float16 or bfloat16, got ",
                t.scalar_type());
    return t.scalar_type() == at::kHalf ? KVMIG_F16 : KVMIG_BF16;
}

// [num_rows, num_heads, head_dim] with a contiguous last dimension.
kvmig_rows rows_of(const at::Tensor& t, const at::Tensor& like, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
    TORCH_CHECK(t.device() == like.device(), name, " is on another device");
    TORCH_CHECK(t.dim() == 3, name, " must have 3 dimensions [num_rows, num_heads, head_dim], got ", t.dim());
    TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, name, ": the values of a head must be contiguous");
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " differs in dtype");
    kvmig_rows r;
    r.data = t.data_ptr();
    r.num_heads = t.size(1);
    // the stride of a dimension of one element says nothing
    r.row_stride = t.size(0) > 1 ? t.stride(0) : 0;
    r.head_stride = t.size(1) > 1 ? t.stride(1) : 0;
    return r;
}

const int32_t* ints_of(const at::Tensor& t, const at::Tensor& like, int64_t dims, const char* name) {
    TORCH_CHECK(t.device() == like.device(), name, " is on another device");
    TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
    TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimension(s), got ", t.dim());
    TORCH_CHECK(t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1, name, ": the last dimension must be contiguous");
    return t.const_data_ptr<int32_t>();
}

kvmig_batch batch_of(const at::Tensor& like, const at::Tensor& starts, const at::Tensor* seq_lens, const at::Tensor* block_tables,
                     int64_t max_rows) {
    kvmig_batch b = {};
    b.starts = ints_of(starts, like, 1, "starts");
    TORCH_CHECK(starts.size(0) >= 1, "starts must have one entry more than there are sequences");
    b.num_seqs = starts.size(0) - 1;
    b.num_rows = like.size(0);
    b.max_rows = max_rows;
    if (seq_lens) {
        b.seq_lens = ints_of(*seq_lens, like, 1, "seq_lens");
        TORCH_CHECK(seq_lens->size(0) == b.num_seqs, "seq_lens has ", seq_lens->size(0), " entries for ", b.num_seqs, " sequences");
    }
    if (block_tables) {
        b.block_tables = ints_of(*block_tables, like, 2, "block_tables");
        TORCH_CHECK(block_tables->size(0) == b.num_seqs, "block_tables has ", block_tables->size(0), " rows for ", b.num_seqs, " sequences");
        b.max_blocks = block_tables->size(1);
        b.table_stride = b.num_seqs > 1 ? block_tables->stride(0) : b.max_blocks;
    }
    return b;
}

// Shape of the pools.  Their element type is the rows' own, or uint8 for quantised pools.
kvmig_pool_shape pools_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& rows) {
    TORCH_CHECK(k.is_cuda() && v.is_cuda(), "k_cache and v_cache must be CUDA tensors");
    TORCH_CHECK(k.dim() == 5, "k_cache must have 5 dimensions [num_blocks, num_layers, num_heads, block_size, head_dim], got ", k.dim());
    TORCH_CHECK(k.sizes() == v.sizes(), "k_cache and v_cache differ in shape");
    TORCH_CHECK(k.scalar_type() == v.scalar_type(), "k_cache and v_cache differ in dtype");
    TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), "k_cache and v_cache must be contiguous");
    TORCH_CHECK(k.device() == rows.device() && v.device() == rows.device(), "the pools are on another device than the rows");
    const bool quantised = k.scalar_type() == at::kByte;
    TORCH_CHECK(quantised || k.scalar_type() == rows.scalar_type(), "pools of ", k.scalar_type(), " do not hold rows of ",
                rows.scalar_type(), ": they have the rows' type, or are uint8 for quantised pools");
    TORCH_CHECK(rows.dim() == 3 && rows.size(2) + (quantised ? KVMIG_SCALE_BYTES : 0) == k.size(4), "the last dimension of the pools is ",
                k.size(4), " and of the rows ", rows.size(rows.dim() - 1),
                quantised ? ": a quantised pool has 4 bytes more than head_dim" : "");
    return kvmig_pool_shape{k.size(0), k.size(1), k.size(2), k.size(3), k.size(4), static_cast<int64_t>(k.element_size())};
}

// The operators compute no gradients: a call that autograd would have to follow, backward or forward, is refused rather than cut
// off silently.
void check_no_grad(std::initializer_list<const at::Tensor*> inputs, const char* op) {
    for (const at::Tensor* t : inputs)
        TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), op, " has no gradient, and an argument carries a forward-mode tangent");
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor* t : inputs) TORCH_CHECK(!t->requires_grad(), op, " has no gradient: call it under torch.no_grad()");
}

void check_written(const at::Tensor& t, std::initializer_list<const at::Tensor*> others, const char* name) {
    at::assert_no_internal_overlap(t);
    for (const at::Tensor* o : others)
        if (t.numel() && o->numel()) at::assert_no_overlap(t, *o);
}

// The call has been enqueued: autograd takes note that these were overwritten.  (Tensors made in inference mode keep no count.)
void count_written(std::initializer_list<const at::Tensor*> written) {
    for (const at::Tensor* t : written)
        if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// kv_cache_ops::write
void write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache, int64_t layer,
           const at::Tensor& block_tables, const at::Tensor& seq_lens, const at::Tensor& starts) {
    check_no_grad({&k, &v, &k_cache, &v_cache}, "write");
    const int dtype = dtype_of(k, "k");
    const kvmig_rows kr = rows_of(k, k, "k"), vr = rows_of(v, k, "v");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v differ in shape");
    const kvmig_pool_shape s = pools_of(k_cache, v_cache, k);
    const kvmig_batch b = batch_of(k, starts, &seq_lens, &block_tables, k.size(0));
    check_written(k_cache, {&v_cache, &k, &v}, "k_cache");
    check_written(v_cache, {&k, &v}, "v_cache");
    c10::cuda::CUDAGuard guard(k.device());
    check(kvmig_cache_write(&kr, &vr, dtype, k_cache.data_ptr(), v_cache.data_ptr(), &s, layer, &b,
                            c10::cuda::getCurrentCUDAStream(k.device().index()).stream()),
          "write");
    count_written({&k_cache, &v_cache});
}

// kv_cache_ops::read
void read(const at::Tensor& k_cache, const at::Tensor& v_cache, int64_t layer, const at::Tensor& block_tables, const at::Tensor& starts,
          const at::Tensor& k_out, const at::Tensor& v_out) {
    check_no_grad({&k_out, &v_out, &k_cache, &v_cache}, "read");
    const int dtype = dtype_of(k_out, "k_out");
    const kvmig_rows kr = rows_of(k_out, k_out, "k_out"), vr = rows_of(v_out, k_out, "v_out");
    TORCH_CHECK(k_out.sizes() == v_out.sizes(), "k_out and v_out differ in shape");
    const kvmig_pool_shape s = pools_of(k_cache, v_cache, k_out);
    const kvmig_batch b = batch_of(k_out, starts, nullptr, &block_tables, k_out.size(0));
    check_written(k_out, {&v_out, &k_cache, &v_cache}, "k_out");
    check_written(v_out, {&k_cache, &v_cache}, "v_out");
    c10::cuda::CUDAGuard guard(k_out.device());
    check(kvmig_cache_read(k_cache.data_ptr(), v_cache.data_ptr(), &s, layer, &b, &kr, &vr, dtype,
                           c10::cuda::getCurrentCUDAStream(k_out.device().index()).stream()),
          "read");
    count_written({&k_out, &v_out});
}

// kv_attention_ops::paged
void paged(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache, int64_t layer, const at::Tensor& block_tables,
           const at::Tensor& seq_lens, const at::Tensor& starts, int64_t max_rows, double scale, const at::Tensor& out) {
    check_no_grad({&q, &k_cache, &v_cache, &out}, "paged");
    const int dtype = dtype_of(q, "q");
    const kvmig_rows qr = rows_of(q, q, "q"), orow = rows_of(out, q, "out");
    TORCH_CHECK(q.sizes() == out.sizes(), "q and out differ in shape");
    const kvmig_pool_shape s = pools_of(k_cache, v_cache, q);
    const kvmig_batch b = batch_of(q, starts, &seq_lens, &block_tables, max_rows);
    check_written(out, {&q, &k_cache, &v_cache}, "out");
    c10::cuda::CUDAGuard guard(q.device());
    const int64_t bytes = kvmig_paged_attention_workspace(&s, qr.num_heads, &b);
    check(bytes, "paged");
    at::Tensor workspace;
    if (bytes > 0) workspace = at::empty({bytes}, q.options().dtype(at::kByte));
    check(kvmig_paged_attention(&qr, &orow, dtype, k_cache.data_ptr(), v_cache.data_ptr(), &s, layer, &b, scale,
                                bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                                c10::cuda::getCurrentCUDAStream(q.device().index()).stream()),
          "paged");
    count_written({&out});
}

// kv_attention_ops::prompt
void prompt(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& starts, int64_t max_rows, double scale,
            const at::Tensor& out) {
    check_no_grad({&q, &k, &v, &out}, "prompt");
    const int dtype = dtype_of(q, "q");
    const kvmig_rows qr = rows_of(q, q, "q"), kr = rows_of(k, q, "k"), vr = rows_of(v, q, "v"), orow = rows_of(out, q, "out");
    TORCH_CHECK(q.sizes() == out.sizes(), "q and out differ in shape");
    TORCH_CHECK(k.sizes() == v.sizes(), "k and v differ in shape");
    TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2), "q and k differ in rows or head_dim");
    const kvmig_batch b = batch_of(q, starts, nullptr, nullptr, max_rows);
    check_written(out, {&q, &k, &v}, "out");
    c10::cuda::CUDAGuard guard(q.device());
    check(kvmig_prompt_attention(&qr, &kr, &vr, &orow, dtype, q.size(2), &b, scale,
                                 c10::cuda::getCurrentCUDAStream(q.device().index()).stream()),
          "prompt");
    count_written({&out});
}

}  // namespace

TORCH_LIBRARY(kv_cache_ops, m) {
    m.def("write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, int layer, Tensor block_tables, Tensor seq_lens, "
          "Tensor starts) -> ()",
          &write);
    m.def("read(Tensor k_cache, Tensor v_cache, int layer, Tensor block_tables, Tensor starts, Tensor(a!) k_out, Tensor(b!) v_out) -> ()",
          &read);
}

TORCH_LIBRARY(kv_attention_ops, m) {
    m.def("paged(Tensor q, Tensor k_cache, Tensor v_cache, int layer, Tensor block_tables, Tensor seq_lens, Tensor starts, "
          "int max_rows, float scale, Tensor(a!) out) -> ()",
          &paged);
    m.def("prompt(Tensor q, Tensor k, Tensor v, Tensor starts, int max_rows, float scale, Tensor(a!) out) -> ()", &prompt);
}
