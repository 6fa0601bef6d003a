// Python bindings of the token-by-token operators (csrc/ops/serving.hpp).  Every function checks its operands, allocates outputs and
// workspaces through torch and launches on the current CUDA stream of the operands' device, so the calls can be captured in a CUDA graph.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <limits>

#include "../core/errors.hpp"
#include "../ops/ops.hpp"
#include "../ops/serving.hpp"
#include "bind.hpp"
#include "operand_checks.hpp"

namespace py = pybind11;

namespace mccl {

namespace {

struct Cache {
  ops::PagedTensor k, v;
  ops::PageTable table;
  int kv_heads, head_dim;
};
Cache cache_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& like, const char* op) {
  for (const auto* t : {&k, &v}) {
    need_on(*t, like, op);
    MCCL_CHECK_TENSOR(t->dim() == 4, op << ": pages must be [pages, kv_heads, page_size, head_dim]");
    MCCL_CHECK_TENSOR(t->scalar_type() == like.scalar_type(), op << ": pages of dtype " << c10::toString(t->scalar_type()) << " with "
                                                                 << c10::toString(like.scalar_type()));
    MCCL_CHECK_TENSOR(vector_rows(*t), op << ": pages need a contiguous head_dim, strides that are multiples of 8 and a 16-byte aligned base");
  }
  MCCL_CHECK_TENSOR(k.sizes() == v.sizes(), op << ": keys and values of different sizes");
  MCCL_CHECK_TENSOR(k.size(2) > 0, op << ": page_size must be positive");
  need_on(table, like, op);
  MCCL_CHECK_TENSOR(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
                    op << ": the page table must be int32 [sequences, pages] with contiguous rows");
  Cache c;
  c.k = {k.data_ptr(), k.stride(0), k.stride(1), k.stride(2)};
  c.v = {v.data_ptr(), v.stride(0), v.stride(1), v.stride(2)};
  c.table.p = table.data_ptr<int>();
  c.table.stride = table.stride(0);
  c.table.rows = as_int(table.size(0), op);
  c.table.width = as_int(table.size(1), op);
  c.table.page_size = as_int(k.size(2), op);
  c.table.pages = as_int(k.size(0), op);
  // positions are counted in 32 bits, rounded up to whole tiles
  MCCL_CHECK_TENSOR(static_cast<int64_t>(c.table.width) * c.table.page_size <= std::numeric_limits<int>::max() - 64,
                    op << ": a row of the page table holds more than 2^31 - 65 positions");
  c.kv_heads = as_int(k.size(1), op);
  c.head_dim = as_int(k.size(3), op);
  return c;
}
// A 4-bit weight as the kernels read it: 16 bytes of codes and 8 of parameters at a time.
void need_w4(const at::Tensor& codes, const at::Tensor& params, int64_t n, int64_t k, int64_t group, const char* op) {
  MCCL_CHECK_TENSOR((group == 32 || group == 64 || group == 128 || group == 256) && n >= 0 && k >= 0 && k % group == 0 && codes.is_contiguous() && params.is_contiguous() &&
                        codes.numel() * static_cast<int64_t>(codes.element_size()) == (n + 15) / 16 * ((k + 63) / 64) * 512 && params.scalar_type() == at::kInt &&
                        params.numel() == (n + 15) / 16 * (k / group) * 16,
                    op << ": the weight is not laid out for [" << n << ", " << k << "]");
  MCCL_CHECK_TENSOR(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(params.data_ptr()) % 8 == 0,
                    op << ": codes must begin on a 16-byte boundary, parameters on one of 8 bytes");
}

}  // namespace

void bind_serving(py::module_& m) {
  m.def(
      "paged_append",
      [](const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
         const at::Tensor& positions, const c10::optional<at::Tensor>& rows, const c10::optional<at::Tensor>& q,
         const c10::optional<at::Tensor>& cos_t, const c10::optional<at::Tensor>& sin_t) -> c10::optional<at::Tensor> {
        const char* op = "paged_append";
        need_on(k, k, op);
        need_on(v, k, op);
        for (const auto* t : {&k, &v, &k_pages, &v_pages}) need_forward_only(*t, op);
        ops::AppendArgs a;
        a.type = half16(k, op);
        MCCL_CHECK_TENSOR(v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes(), op << ": k and v differ in dtype or sizes");
        const Cache c = cache_of(k_pages, v_pages, table, k, op);
        MCCL_CHECK_TENSOR(!repeated(k_pages) && !repeated(v_pages) && !same_memory(k_pages, v_pages), op << ": pages that overlap in memory");
        a.k = tokens_of(k, "paged_append(k)");
        a.v = tokens_of(v, "paged_append(v)");
        a.k_pages = c.k;
        a.v_pages = c.v;
        a.table = c.table;
        a.tokens = k.size(0);
        a.kv_heads = c.kv_heads;
        a.head_dim = c.head_dim;
        MCCL_CHECK_TENSOR(k.size(1) == c.kv_heads && k.size(2) == c.head_dim, op << ": k has other heads or another head_dim than the cache");
        MCCL_CHECK_TENSOR(c.head_dim % 8 == 0 && c.head_dim > 0, op << ": head_dim must be a positive multiple of 8");
        a.positions = need_int32(positions, k, a.tokens, "paged_append(positions)");
        if (rows.has_value()) a.rows = need_int32(*rows, k, a.tokens, "paged_append(rows)");
        MCCL_CHECK_TENSOR(cos_t.has_value() == sin_t.has_value(), op << ": cos and sin come together");
        MCCL_CHECK_TENSOR(!q.has_value() || cos_t.has_value(), op << ": q is only taken to be rotated, and there are no rotation tables");
        if (cos_t.has_value()) {
          for (const auto* t : {&*cos_t, &*sin_t}) {
            need_on(*t, k, "paged_append(rope)");
            need_forward_only(*t, op);
            MCCL_CHECK_TENSOR(t->scalar_type() == at::kFloat && t->dim() == 2 && t->is_contiguous() && t->size(1) * 2 == c.head_dim &&
                                  reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                              "paged_append(rope): cos and sin must be contiguous fp32 [positions, head_dim / 2]");
          }
          MCCL_CHECK_TENSOR(cos_t->sizes() == sin_t->sizes(), "paged_append(rope): cos and sin of different sizes");
          a.cos = cos_t->data_ptr<float>();
          a.sin = sin_t->data_ptr<float>();
          a.rope_rows = as_int(cos_t->size(0), op);
        }
        c10::cuda::CUDAGuard guard(k.device());
        c10::optional<at::Tensor> out;
        if (q.has_value()) {
          need_on(*q, k, "paged_append(q)");
          need_forward_only(*q, op);
          a.q = tokens_of(*q, "paged_append(q)");
          MCCL_CHECK_TENSOR(q->scalar_type() == k.scalar_type() && q->size(0) == a.tokens && q->size(2) == c.head_dim,
                            "paged_append(q): another dtype, other tokens or another head_dim than k");
          a.heads = as_int(q->size(1), op);
          out = empty_on(k, {a.tokens, q->size(1), q->size(2)}, k.scalar_type());
          a.q_out = out->data_ptr();
        }
        check_launch(ops::paged_append(a, stream_of(k)), op);
        return out;
      },
      py::arg("k"), py::arg("v"), py::arg("k_pages"), py::arg("v_pages"), py::arg("table"), py::arg("positions"), py::arg("rows") = py::none(),
      py::arg("q") = py::none(), py::arg("cos") = py::none(), py::arg("sin") = py::none());

  m.def(
      "copy_pages",
      [](at::Tensor pages, const at::Tensor& src, const at::Tensor& dst, int64_t dim) {
        const char* op = "copy_pages";
        need_on(pages, pages, op);
        need_forward_only(pages, op);
        if (dim < 0) dim += pages.dim();
        MCCL_CHECK_TENSOR(dim >= 0 && dim < pages.dim(), op << ": dim out of range");
        MCCL_CHECK_TENSOR(src.dim() == 1, op << ": src must be one-dimensional");
        const int* s = need_int32(src, pages, src.numel(), "copy_pages(src)");
        const int* d = need_int32(dst, pages, src.numel(), "copy_pages(dst)");
        const int64_t item = static_cast<int64_t>(pages.element_size());
        // a page is one run of memory; the dimensions before it are one dimension
        int64_t page = 1;
        for (int64_t i = pages.dim() - 1; i > dim; --i) {
          MCCL_CHECK_TENSOR(pages.size(i) <= 1 || pages.stride(i) == page, op << ": a page must be contiguous");
          page *= pages.size(i);
        }
        int64_t outer = 1, outer_stride = 0;
        for (int64_t i = dim - 1; i >= 0; --i) {
          if (pages.size(i) == 1) continue;
          if (outer == 1) outer_stride = pages.stride(i);
          MCCL_CHECK_TENSOR(pages.stride(i) == outer_stride * outer, op << ": the dimensions before the pages must have one common stride");
          outer *= pages.size(i);
        }
        // pages of one outer index lie one after the other and the outer indices behind them, or the outer indices within a page's stride
        const int64_t many = pages.size(dim), stride = pages.stride(dim);
        MCCL_CHECK_TENSOR((many <= 1 || stride >= page) && (outer <= 1 || (outer_stride >= page && (many <= 1 || outer_stride >= (many - 1) * stride + page ||
                                                                                                   stride >= (outer - 1) * outer_stride + page))),
                          op << ": pages that overlap in memory");
        const int count = as_int(pages.size(dim), op);
        c10::cuda::CUDAGuard guard(pages.device());
        if (pages.numel() > 0)
          check_launch(ops::copy_pages(pages.data_ptr(), outer, outer_stride * item, pages.stride(dim) * item, page * item, count, s, d, src.numel(),
                                       stream_of(pages)),
                       op);
        return pages;
      },
      py::arg("pages"), py::arg("src"), py::arg("dst"), py::arg("dim") = 0);

  m.def(
      "paged_attention",
      [](const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table, const at::Tensor& lengths, double scale,
         int64_t window, int64_t sinks, bool return_lse) {
        const char* op = "paged_attention";
        need_on(q, q, op);
        for (const auto* t : {&q, &k_pages, &v_pages}) need_forward_only(*t, op);
        ops::PagedAttentionArgs a;
        a.type = half16(q, op);
        const Cache c = cache_of(k_pages, v_pages, table, q, op);
        a.q = tokens_of(q, "paged_attention(q)");
        a.k_pages = c.k;
        a.v_pages = c.v;
        a.table = c.table;
        a.batch = as_int(q.size(0), op);
        a.heads = as_int(q.size(1), op);
        a.kv_heads = c.kv_heads;
        a.head_dim = c.head_dim;
        MCCL_CHECK_TENSOR(q.size(2) == c.head_dim, op << ": q has head_dim " << q.size(2) << ", the cache " << c.head_dim);
        MCCL_CHECK_TENSOR(c.head_dim % 8 == 0 && c.head_dim > 0 && c.head_dim <= 256, op << ": head_dim must be a multiple of 8 up to 256");
        MCCL_CHECK_TENSOR(c.kv_heads > 0 && a.heads % c.kv_heads == 0, op << ": " << a.heads << " query heads over " << c.kv_heads << " heads of keys and values");
        MCCL_CHECK_TENSOR(c.table.rows == a.batch, op << ": a page table of " << c.table.rows << " rows for " << a.batch << " sequences");
        MCCL_CHECK_TENSOR(sinks >= 0, op << ": sinks must not be negative");
        a.lengths = need_int32(lengths, q, a.batch, "paged_attention(lengths)");
        a.scale = static_cast<float>(scale);
        const int64_t most = std::numeric_limits<int>::max();
        a.window = static_cast<int>(std::min(window, most));
        a.sinks = static_cast<int>(std::min(sinks, most));
        c10::cuda::CUDAGuard guard(q.device());
        at::Tensor o = empty_on(q, {q.size(0), q.size(1), q.size(2)}, q.scalar_type());
        c10::optional<at::Tensor> lse;
        a.o = o.data_ptr();
        if (return_lse) {
          lse = empty_on(q, {q.size(0), q.size(1)}, at::kFloat);
          a.lse = lse->data_ptr<float>();
        }
        at::Tensor workspace;
        if (const size_t bytes = ops::paged_attention_workspace(a)) {
          workspace = empty_on(q, {static_cast<int64_t>(bytes)}, at::kByte);
          a.workspace = workspace.data_ptr();
        }
        check_launch(ops::paged_attention(a, stream_of(q)), op);
        return std::make_pair(o, lse);
      },
      py::arg("q"), py::arg("k_pages"), py::arg("v_pages"), py::arg("table"), py::arg("lengths"), py::arg("scale"), py::arg("window") = 0,
      py::arg("sinks") = 0, py::arg("return_lse") = false);

  m.def(
      "w4_linear",
      [](const at::Tensor& x, const at::Tensor& codes, const at::Tensor& params, int64_t n, int64_t k, int64_t group, const c10::optional<at::Tensor>& bias,
         bool gelu, const c10::optional<at::Tensor>& residual) {
        const char* op = "linear_w4";
        need_on(x, x, op);
        need_on(codes, x, op);
        need_on(params, x, op);
        need_forward_only(x, op);
        MCCL_CHECK_TENSOR(x.scalar_type() == at::kBFloat16, op << ": expected bf16, got " << c10::toString(x.scalar_type()));
        MCCL_CHECK_TENSOR(x.dim() >= 1 && x.size(-1) == k, op << ": x must have " << k << " columns");
        need_w4(codes, params, n, k, group, op);
        c10::cuda::CUDAGuard guard(x.device());
        at::Tensor x2 = x.dim() == 2 ? x : x.reshape({-1, k});
        if (!vector_rows(x2)) x2 = x2.clone(at::MemoryFormat::Contiguous);
        ops::W4Args a;
        a.x = x2.data_ptr();
        a.ldx = x2.stride(0);
        a.codes = codes.data_ptr();
        a.params = params.data_ptr();
        a.m = as_int(x2.size(0), op);
        a.n = as_int(n, op);
        a.k = as_int(k, op);
        a.group = as_int(group, op);
        a.gelu = gelu;
        at::Tensor bias_f, res2;
        if (bias.has_value()) {
          need_on(*bias, x, "linear_w4(bias)");
          need_forward_only(*bias, op);
          MCCL_CHECK_TENSOR(bias->dim() == 1 && bias->numel() == n && bias->scalar_type() == at::kFloat && bias->is_contiguous(),
                            "linear_w4(bias): expected contiguous fp32 [" << n << "]");
          a.bias = bias->data_ptr<float>();
        }
        at::DimVector shape(x.sizes().begin(), x.sizes().end());
        shape.back() = n;
        if (residual.has_value()) {
          need_on(*residual, x, "linear_w4(residual)");
          need_forward_only(*residual, op);
          MCCL_CHECK_TENSOR(residual->scalar_type() == at::kBFloat16 && residual->sizes() == at::IntArrayRef(shape.data(), shape.size()),
                            "linear_w4(residual): expected bf16 of the output's shape");
          res2 = residual->dim() == 2 ? *residual : residual->reshape({-1, n});
          if (res2.size(1) > 1 && res2.stride(1) != 1) res2 = res2.contiguous();
          a.residual = res2.data_ptr();
          a.ldr = res2.stride(0);
        }
        at::Tensor y = empty_on(x, shape, at::kBFloat16);
        a.y = y.data_ptr();
        check_launch(ops::w4_linear(a, stream_of(x)), op);
        return y;
      },
      py::arg("x"), py::arg("codes"), py::arg("params"), py::arg("n"), py::arg("k"), py::arg("group"), py::arg("bias") = py::none(),
      py::arg("gelu") = false, py::arg("residual") = py::none());

  m.def(
      "w4_pack",
      [](at::Tensor codes, const at::Tensor& scales, const c10::optional<at::Tensor>& zeros) {
        const char* op = "w4_pack";
        need_on(codes, codes, op);
        need_on(scales, codes, op);
        MCCL_CHECK_TENSOR(codes.scalar_type() == at::kByte && codes.dim() == 2 && codes.is_contiguous(), op << ": codes must be contiguous uint8 [n, k]");
        const int64_t n = codes.size(0), k = codes.size(1);
        MCCL_CHECK_TENSOR(scales.scalar_type() == at::kBFloat16 && scales.dim() == 2 && scales.is_contiguous() && scales.size(0) == n && scales.size(1) > 0 && k % scales.size(1) == 0 &&
                              k / scales.size(1) % 32 == 0,
                          op << ": scales must be contiguous bf16 [n, groups]");
        if (zeros.has_value()) {
          need_on(*zeros, codes, op);
          MCCL_CHECK_TENSOR(zeros->scalar_type() == at::kByte && zeros->is_contiguous() && zeros->sizes() == scales.sizes(), op << ": zeros must be contiguous uint8 of the scales' shape");
        }
        c10::cuda::CUDAGuard guard(codes.device());
        // the kernel reads two codes at a time: k is even, and codes that begin on an odd byte (a part of a buffer) are moved first
        if (reinterpret_cast<uintptr_t>(codes.data_ptr()) % 2 != 0) codes = codes.clone();
        const int64_t tiles = (n + 15) / 16;
        at::Tensor packed = empty_on(codes, {tiles, (k + 63) / 64, 32, 16}, at::kByte), params = empty_on(codes, {tiles, scales.size(1), 8, 2}, at::kInt);
        at::Tensor bad = at::zeros({1}, codes.options().dtype(at::kInt));
        check_launch(ops::w4_pack(codes.data_ptr<uint8_t>(), scales.data_ptr(), zeros.has_value() ? zeros->data_ptr<uint8_t>() : nullptr, packed.data_ptr(), params.data_ptr(),
                                  bad.data_ptr<int>(), as_int(n, op), as_int(k, op), as_int(k / scales.size(1), op), stream_of(codes)),
                     op);
        return std::make_tuple(packed, params, bad);
      },
      py::arg("codes"), py::arg("scales"), py::arg("zeros") = py::none());

  m.def(
      "w4_dequantize",
      [](const at::Tensor& codes, const at::Tensor& params, int64_t n, int64_t k, int64_t group) {
        need_on(codes, codes, "w4_dequantize");
        need_on(params, codes, "w4_dequantize");
        need_w4(codes, params, n, k, group, "w4_dequantize");
        c10::cuda::CUDAGuard guard(codes.device());
        at::Tensor w = empty_on(codes, {n, k}, at::kBFloat16);
        check_launch(ops::w4_dequantize(codes.data_ptr(), params.data_ptr(), w.data_ptr(), as_int(n, "w4_dequantize"), as_int(k, "w4_dequantize"),
                                        as_int(group, "w4_dequantize"), stream_of(codes)),
                     "w4_dequantize");
        return w;
      },
      py::arg("codes"), py::arg("params"), py::arg("n"), py::arg("k"), py::arg("group"));
}

}  // namespace mccl
