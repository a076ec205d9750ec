// at::Tensor shim over the C ABI of include/pulsar_paged.h and its torch
// registration, in the manner of torch_ops.cpp.
#include "pulsar_paged_ops.hpp"

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <cmath>

#include "pulsar_paged.h"

namespace pulsar {
namespace {

using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;

pw4_stream_t current_stream() {
    return reinterpret_cast<pw4_stream_t>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
}

void check_status(int rc, const char* op) {
    if (rc == PW4_ERR_HIP) {
        TORCH_CHECK(false, op, ": ", pw4_status_string(rc), ": ", pw4_last_hip_error());
    }
    TORCH_CHECK(rc == PW4_OK, op, ": ", pw4_status_string(rc));
}

// at::empty on like's device without the dispatcher's way there: a call of the small
// operators is as long as its host side, and some have six outputs.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}

at::Tensor scratch(size_t bytes, const at::Tensor& like) {
    return fresh({(int64_t)std::max<size_t>(bytes, 16)}, at::kByte, like);
}

void check_device(const char* op, const at::Tensor& first, std::initializer_list<const at::Tensor*> others) {
    TORCH_CHECK(first.is_cuda(), op, ": all inputs must be CUDA tensors");
    for (const at::Tensor* t : others) {
        TORCH_CHECK(t->is_cuda() && t->device() == first.device(), op, ": all inputs must be on one CUDA device");
    }
}

void check_ints(const char* op, const char* name, const at::Tensor& t, int64_t dim, at::ScalarType type = at::kInt) {
    TORCH_CHECK(t.scalar_type() == type && t.dim() == dim, op, ": ", name, " must be ",
                type == at::kInt ? "int32" : "int64", " and ", dim, "-D");
    TORCH_CHECK(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, op, ": ", name,
                " must be contiguous in its last dimension");
}

// The book-keeping of a pool: int32 ref_counts [P], block_tables [rows, width], seq_lens [rows].
void check_tables(const char* op, const at::Tensor* refs, const at::Tensor& tables, const at::Tensor* lens) {
    if (refs) check_ints(op, "ref_counts", *refs, 1);
    check_ints(op, "block_tables", tables, 2);
    TORCH_CHECK(tables.numel() == 0 || tables.size(0) == 1 || tables.stride(0) >= tables.size(1), op,
                ": block_tables' rows overlap");
    if (lens) {
        check_ints(op, "seq_lens", *lens, 1);
        TORCH_CHECK(lens->size(0) == tables.size(0), op, ": seq_lens must be [rows of block_tables]");
    }
}

int64_t table_stride(const at::Tensor& tables) {
    return tables.size(0) > 1 ? tables.stride(0) : std::max<int64_t>(tables.size(1), 1);
}

// A cache [P, page, heads, dim] as it is used in place: head_dim contiguous.
void check_cache(const char* op, const char* name, const at::Tensor& c) {
    TORCH_CHECK(c.dim() == 4, op, ": ", name, " must be 4-D [pages, page_size, kv_heads, head_dim]");
    TORCH_CHECK(c.numel() == 0 || c.size(3) == 1 || c.stride(3) == 1, op, ": ", name,
                " must be contiguous in its last dimension");
}


void check_half(const char* op, const char* name, const at::Tensor& t) {
    TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, op, ": ", name,
                " must be fp16 or bf16");
}

// Stride of a dimension; that of a dimension of one counts for nothing.
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void check_same_layout(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache) {
    bool same = k_cache.sizes() == v_cache.sizes() && k_cache.scalar_type() == v_cache.scalar_type();
    for (int64_t d = 0; same && d < k_cache.dim(); ++d) same = stride_of(k_cache, d) == stride_of(v_cache, d);
    TORCH_CHECK(same, op, ": k_cache and v_cache must have one shape, dtype and layout");
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

pw4_page_pool as_pool(const char* op, const at::Tensor& pool) {
    TORCH_CHECK(pool.is_cuda(), op, ": all inputs must be CUDA tensors");
    TORCH_CHECK(pool.dim() >= 3, op, ": pool must be [planes, pages, page_size, ...]");
    int64_t elements = 1;
    for (int64_t d = pool.dim() - 1; d >= 2; --d) {
        TORCH_CHECK(pool.numel() == 0 || pool.size(d) == 1 || pool.stride(d) == elements, op,
                    ": pool's pages must be contiguous");
        elements *= pool.size(d);
    }
    const int64_t e = pool.element_size();
    TORCH_CHECK(pool.numel() == 0 || pool.size(1) == 1 || pool.stride(1) >= elements, op, ": pool's pages overlap");
    return pw4_page_pool{pool.data_ptr(), pool.size(0), pool.size(1), elements * e, stride_of(pool, 0) * e,
                         stride_of(pool, 1) * e};
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> paged_attention_cuda(const at::Tensor& q, const at::Tensor& k_cache,
                                                        const at::Tensor& v_cache, const at::Tensor& block_tables,
                                                        const at::Tensor& seq_lens, const at::Tensor& cu_q,
                                                        int64_t max_q_len, int64_t max_seq_len,
                                                        std::optional<double> scale, int64_t window, double softcap,
                                                        bool return_lse) {
    const char* const op = "paged_attention";
    check_device(op, q, {&k_cache, &v_cache, &block_tables, &seq_lens, &cu_q});
    check_half(op, "q", q);
    TORCH_CHECK(q.dim() == 3, op, ": q must be 3-D [T, q_heads, head_dim]");
    check_cache(op, "k_cache", k_cache);
    check_cache(op, "v_cache", v_cache);
    check_same_layout(op, k_cache, v_cache);
    TORCH_CHECK(k_cache.scalar_type() == q.scalar_type(), op, ": q and the caches must have one dtype");
    check_tables(op, nullptr, block_tables, &seq_lens);
    check_ints(op, "cu_q", cu_q, 1);
    const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), B = block_tables.size(0), Hkv = k_cache.size(2);
    TORCH_CHECK(cu_q.size(0) == B + 1, op, ": cu_q must be [batch + 1]");
    TORCH_CHECK(k_cache.size(3) == D, op, ": q and the caches differ in head_dim");
    TORCH_CHECK(D > 0 && D <= 256 && D % 8 == 0, op, ": head_dim must be a multiple of 8 up to 256");
    TORCH_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, op, ": q_heads must be a multiple of kv_heads");
    TORCH_CHECK(k_cache.size(1) > 0, op, ": page_size must be positive");
    TORCH_CHECK(max_q_len >= 0 && max_seq_len >= 0, op, ": max_q_len and max_seq_len must not be negative");
    TORCH_CHECK(window >= 0, op, ": window must not be negative");
    TORCH_CHECK(softcap >= 0 && std::isfinite((float)softcap), op, ": softcap must be finite in fp32 and not negative");
    TORCH_CHECK(!scale || std::isfinite((float)*scale), op, ": scale must be finite in fp32");
    for (const at::Tensor* c : {&k_cache, &v_cache}) {
        TORCH_CHECK(c->numel() == 0 || (aligned16(*c) && stride_of(*c, 0) % 8 == 0 && stride_of(*c, 1) % 8 == 0 &&
                                        stride_of(*c, 2) % 8 == 0),
                    op, ": the caches' rows must be 16-byte aligned");
    }
    DeviceGuard guard(q.device());
    // q is a slice of a fused projection as often as not: it is read in place where 16-byte loads can
    const bool in_place = q.numel() == 0 || (q.stride(2) == 1 && aligned16(q) && stride_of(q, 0) % 8 == 0 &&
                                             stride_of(q, 1) % 8 == 0);
    const at::Tensor qc = in_place ? q : q.contiguous();
    at::Tensor out = fresh({T, Hq, D}, q.scalar_type(), q);
    at::Tensor lse = fresh({return_lse ? T : 0, Hq}, at::kFloat, q);
    if (T == 0) return {out, lse};
    pw4_paged_attention_args a{};
    a.q = qc.data_ptr();
    a.k_cache = k_cache.data_ptr();
    a.v_cache = v_cache.data_ptr();
    a.block_tables = block_tables.data_ptr<int32_t>();
    a.seq_lens = seq_lens.data_ptr<int32_t>();
    a.cu_q = cu_q.data_ptr<int32_t>();
    a.out = out.data_ptr();
    a.lse = return_lse ? lse.data_ptr<float>() : nullptr;
    a.num_tokens = T;
    a.batch = B;
    a.q_heads = Hq;
    a.kv_heads = Hkv;
    a.head_dim = D;
    a.num_pages = k_cache.size(0);
    a.page_size = k_cache.size(1);
    a.table_width = block_tables.size(1);
    a.table_stride = table_stride(block_tables);
    a.q_token_stride = stride_of(qc, 0);
    a.q_head_stride = stride_of(qc, 1);
    a.page_stride = stride_of(k_cache, 0);
    a.row_stride = stride_of(k_cache, 1);
    a.kv_head_stride = stride_of(k_cache, 2);
    a.max_q_len = std::min(max_q_len, T);
    a.max_seq_len = max_seq_len;
    a.window = window;
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)D));
    // (a cap above 0 stays one: the kernel takes what is below 2^-100 as 2^-100)
    a.softcap = softcap > 0 ? std::max((float)softcap, 0x1p-100f) : 0.f;
    a.dtype = q.scalar_type() == at::kBFloat16 ? PW4_DTYPE_BF16 : PW4_DTYPE_F16;
    const size_t bytes = pw4_paged_attention_workspace_size(&a);
    const at::Tensor ws = bytes ? scratch(bytes, q) : at::Tensor();
    check_status(pw4_paged_attention(&a, bytes ? ws.data_ptr() : nullptr, bytes, current_stream()), op);
    return {out, lse};
}

std::tuple<at::Tensor, at::Tensor> paged_cache_extend_cuda(at::Tensor& ref_counts, at::Tensor& block_tables,
                                                           at::Tensor& seq_lens, const at::Tensor& cu_q,
                                                           int64_t num_tokens, int64_t page_size) {
    const char* const op = "paged_cache_extend";
    check_device(op, block_tables, {&ref_counts, &seq_lens, &cu_q});
    check_tables(op, &ref_counts, block_tables, &seq_lens);
    check_ints(op, "cu_q", cu_q, 1);
    TORCH_CHECK(cu_q.size(0) == block_tables.size(0) + 1, op, ": cu_q must be [rows + 1]");
    TORCH_CHECK(num_tokens >= 0, op, ": num_tokens must not be negative");
    TORCH_CHECK(page_size > 0, op, ": page_size must be positive");
    DeviceGuard guard(block_tables.device());
    at::Tensor slots = fresh({num_tokens}, at::kLong, block_tables);
    at::Tensor missing = fresh({1}, at::kInt, block_tables);
    check_status(pw4_paged_cache_extend(ref_counts.data_ptr<int32_t>(), ref_counts.size(0),
                                        block_tables.data_ptr<int32_t>(), block_tables.size(1),
                                        table_stride(block_tables), seq_lens.data_ptr<int32_t>(),
                                        cu_q.data_ptr<int32_t>(), block_tables.size(0), num_tokens, page_size,
                                        slots.data_ptr<int64_t>(), missing.data_ptr<int32_t>(), current_stream()),
                 op);
    return {slots, missing};
}

void paged_cache_write_cuda(const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache, at::Tensor& v_cache,
                            const at::Tensor& slots) {
    const char* const op = "paged_cache_write";
    check_device(op, k_cache, {&k, &v, &v_cache, &slots});
    check_cache(op, "k_cache", k_cache);
    check_cache(op, "v_cache", v_cache);
    check_same_layout(op, k_cache, v_cache);
    check_half(op, "k_cache", k_cache);
    check_ints(op, "slots", slots, 1, at::kLong);
    TORCH_CHECK(k.dim() == 3 && v.sizes() == k.sizes(), op, ": k and v must be 3-D [T, kv_heads, head_dim]");
    TORCH_CHECK(k.scalar_type() == k_cache.scalar_type() && v.scalar_type() == k_cache.scalar_type(), op,
                ": k, v and the caches must have one dtype");
    TORCH_CHECK(k.size(0) == slots.size(0), op, ": slots must be [T]");
    TORCH_CHECK(k.size(1) == k_cache.size(2) && k.size(2) == k_cache.size(3), op,
                ": k and the caches differ in kv_heads or head_dim");
    TORCH_CHECK(k_cache.size(1) > 0, op, ": page_size must be positive");
    DeviceGuard guard(k_cache.device());
    const at::Tensor kc = k.size(2) <= 1 || k.stride(2) == 1 ? k : k.contiguous();
    const at::Tensor vc = v.size(2) <= 1 || v.stride(2) == 1 ? v : v.contiguous();
    check_status(pw4_paged_cache_write(kc.data_ptr(), vc.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                       slots.data_ptr<int64_t>(), kc.size(0), kc.size(1), kc.size(2), stride_of(kc, 0),
                                       stride_of(kc, 1), stride_of(vc, 0), stride_of(vc, 1), k_cache.size(0),
                                       k_cache.size(1), stride_of(k_cache, 0), stride_of(k_cache, 1),
                                       stride_of(k_cache, 2), current_stream()),
                 op);
}

void paged_cache_copy_cuda(at::Tensor& pool, const at::Tensor& src_pages, const at::Tensor& dst_pages) {
    const char* const op = "paged_cache_copy";
    const pw4_page_pool p = as_pool(op, pool);
    check_device(op, pool, {&src_pages, &dst_pages});
    check_ints(op, "src_pages", src_pages, 1);
    check_ints(op, "dst_pages", dst_pages, 1);
    TORCH_CHECK(src_pages.size(0) == dst_pages.size(0), op, ": src_pages and dst_pages differ in length");
    DeviceGuard guard(pool.device());
    check_status(pw4_paged_cache_copy(&p, src_pages.data_ptr<int32_t>(), dst_pages.data_ptr<int32_t>(),
                                      src_pages.size(0), current_stream()),
                 op);
}

at::Tensor paged_cache_fork_cuda(at::Tensor& pool, at::Tensor& ref_counts, at::Tensor& block_tables,
                                 at::Tensor& seq_lens, const at::Tensor& src_rows, const at::Tensor& dst_rows) {
    const char* const op = "paged_cache_fork";
    const pw4_page_pool p = as_pool(op, pool);
    check_device(op, pool, {&ref_counts, &block_tables, &seq_lens, &src_rows, &dst_rows});
    check_tables(op, &ref_counts, block_tables, &seq_lens);
    check_ints(op, "src_rows", src_rows, 1);
    check_ints(op, "dst_rows", dst_rows, 1);
    TORCH_CHECK(ref_counts.size(0) == pool.size(1), op, ": ref_counts must be [pages of pool]");
    TORCH_CHECK(src_rows.size(0) == dst_rows.size(0), op, ": src_rows and dst_rows differ in length");
    TORCH_CHECK(pool.size(2) > 0, op, ": page_size must be positive");
    DeviceGuard guard(pool.device());
    at::Tensor missing = fresh({1}, at::kInt, block_tables);
    const size_t bytes = pw4_paged_cache_fork_workspace_size(src_rows.size(0));
    const at::Tensor ws = scratch(bytes, pool);
    check_status(pw4_paged_cache_fork(&p, ref_counts.data_ptr<int32_t>(), block_tables.data_ptr<int32_t>(),
                                      block_tables.size(0), block_tables.size(1), table_stride(block_tables),
                                      seq_lens.data_ptr<int32_t>(), src_rows.data_ptr<int32_t>(),
                                      dst_rows.data_ptr<int32_t>(), src_rows.size(0), pool.size(2),
                                      missing.data_ptr<int32_t>(), ws.data_ptr(), bytes, current_stream()),
                 op);
    return missing;
}

void paged_cache_free_cuda(at::Tensor& ref_counts, at::Tensor& block_tables, at::Tensor& seq_lens,
                           const at::Tensor& rows) {
    const char* const op = "paged_cache_free";
    check_device(op, block_tables, {&ref_counts, &seq_lens, &rows});
    check_tables(op, &ref_counts, block_tables, &seq_lens);
    check_ints(op, "rows", rows, 1);
    DeviceGuard guard(block_tables.device());
    check_status(pw4_paged_cache_free(ref_counts.data_ptr<int32_t>(), ref_counts.size(0),
                                      block_tables.data_ptr<int32_t>(), block_tables.size(0), block_tables.size(1),
                                      table_stride(block_tables), seq_lens.data_ptr<int32_t>(),
                                      rows.data_ptr<int32_t>(), rows.size(0), current_stream()),
                 op);
}

at::Tensor paged_cache_compact_cuda(at::Tensor& pool, at::Tensor& ref_counts, at::Tensor& block_tables) {
    const char* const op = "paged_cache_compact";
    const pw4_page_pool p = as_pool(op, pool);
    check_device(op, pool, {&ref_counts, &block_tables});
    check_tables(op, &ref_counts, block_tables, nullptr);
    TORCH_CHECK(ref_counts.size(0) == pool.size(1), op, ": ref_counts must be [pages of pool]");
    DeviceGuard guard(pool.device());
    at::Tensor used = fresh({1}, at::kInt, block_tables);
    const size_t bytes = pw4_paged_cache_compact_workspace_size(pool.size(1));
    const at::Tensor ws = scratch(bytes, pool);
    check_status(pw4_paged_cache_compact(&p, ref_counts.data_ptr<int32_t>(), block_tables.data_ptr<int32_t>(),
                                         block_tables.size(0), block_tables.size(1), table_stride(block_tables),
                                         used.data_ptr<int32_t>(), ws.data_ptr(), bytes, current_stream()),
                 op);
    return used;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs_cuda(const at::Tensor& logits,
                                                                                           const at::Tensor& targets,
                                                                                           int64_t top_k) {
    const char* const op = "token_logprobs";
    check_device(op, logits, {&targets});
    const auto dt = logits.scalar_type();
    TORCH_CHECK(dt == at::kFloat || dt == at::kHalf || dt == at::kBFloat16, op, ": logits must be fp32, fp16 or bf16");
    TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0, op, ": logits must be 2-D [T, vocab]");
    check_ints(op, "targets", targets, 1, at::kLong);
    TORCH_CHECK(targets.size(0) == logits.size(0), op, ": targets must be [T]");
    TORCH_CHECK(top_k >= 0 && top_k <= 32 && top_k <= logits.size(1), op, ": top_k must be 0 to 32 and at most vocab");
    DeviceGuard guard(logits.device());
    const int64_t T = logits.size(0), V = logits.size(1);
    const at::Tensor x = (V == 1 || logits.stride(1) == 1) && (T <= 1 || logits.stride(0) >= V) ? logits
                                                                                              : logits.contiguous();
    at::Tensor lp = fresh({T}, at::kFloat, logits), ranks = fresh({T}, at::kLong, logits);
    at::Tensor ent = fresh({T}, at::kFloat, logits);
    at::Tensor top = fresh({T, top_k}, at::kFloat, logits), ids = fresh({T, top_k}, at::kLong, logits);
    if (T == 0) return {lp, ranks, ent, top, ids};
    const size_t bytes = pw4_token_logprobs_workspace_size(T, V, top_k);
    const at::Tensor ws = scratch(bytes, logits);
    check_status(pw4_token_logprobs(x.data_ptr(), dt == at::kFloat ? PW4_DTYPE_F32
                                                  : dt == at::kHalf ? PW4_DTYPE_F16
                                                                    : PW4_DTYPE_BF16,
                                    T, V, T > 1 ? x.stride(0) : V, targets.data_ptr<int64_t>(), top_k,
                                    lp.data_ptr<float>(), ranks.data_ptr<int64_t>(), ent.data_ptr<float>(),
                                    top.data_ptr<float>(), ids.data_ptr<int64_t>(), ws.data_ptr(), bytes,
                                    current_stream()),
                 op);
    return {lp, ranks, ent, top, ids};
}

}  // namespace pulsar

TORCH_LIBRARY_FRAGMENT(pulsar, m) {
    m.def(
        "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_tables, Tensor seq_lens, Tensor cu_q, "
        "int max_q_len, int max_seq_len, float? scale=None, int window=0, float softcap=0., bool return_lse=False) "
        "-> (Tensor, Tensor)");
    m.def(
        "paged_cache_extend(Tensor(a!) ref_counts, Tensor(b!) block_tables, Tensor(c!) seq_lens, Tensor cu_q, "
        "int num_tokens, int page_size) -> (Tensor, Tensor)");
    m.def(
        "paged_cache_write(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor slots) -> ()");
    m.def("paged_cache_copy(Tensor(a!) pool, Tensor src_pages, Tensor dst_pages) -> ()");
    m.def(
        "paged_cache_fork(Tensor(a!) pool, Tensor(b!) ref_counts, Tensor(c!) block_tables, Tensor(d!) seq_lens, "
        "Tensor src_rows, Tensor dst_rows) -> Tensor");
    m.def(
        "paged_cache_free(Tensor(a!) ref_counts, Tensor(b!) block_tables, Tensor(c!) seq_lens, Tensor rows) -> ()");
    m.def("paged_cache_compact(Tensor(a!) pool, Tensor(b!) ref_counts, Tensor(c!) block_tables) -> Tensor");
    m.def("token_logprobs(Tensor logits, Tensor targets, int top_k) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(pulsar, CUDA, m) {
    m.impl("paged_attention", TORCH_FN(pulsar::paged_attention_cuda));
    m.impl("paged_cache_extend", TORCH_FN(pulsar::paged_cache_extend_cuda));
    m.impl("paged_cache_write", TORCH_FN(pulsar::paged_cache_write_cuda));
    m.impl("paged_cache_copy", TORCH_FN(pulsar::paged_cache_copy_cuda));
    m.impl("paged_cache_fork", TORCH_FN(pulsar::paged_cache_fork_cuda));
    m.impl("paged_cache_free", TORCH_FN(pulsar::paged_cache_free_cuda));
    m.impl("paged_cache_compact", TORCH_FN(pulsar::paged_cache_compact_cuda));
    m.impl("token_logprobs", TORCH_FN(pulsar::token_logprobs_cuda));
}
