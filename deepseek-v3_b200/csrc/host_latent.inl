// ------------------------------------------------------------------ the 8-bit latent cache (part of host.cpp)
// Planes of a cache: latent e4m3 [pages, page, 512], rope bf16 [pages, page, 64], scale fp32 [pages, page].
struct CachePlanes {
    const at::Tensor &latent, &rope, &scale;
    dsv3_latent_cache_t c;
};

CachePlanes cache_arg(PyObject* latent_o, PyObject* rope_o, PyObject* scale_o) {
    const at::Tensor &latent = tensor_arg(latent_o), &rope = tensor_arg(rope_o), &scale = tensor_arg(scale_o);
    require(latent.is_contiguous() && rope.is_contiguous() && scale.is_contiguous(), "the planes of a cache must be contiguous");
    require(latent.dim() == 3 && rope.dim() == 3 && scale.dim() == 2 && latent.size(2) == DSV3_LATENT_DIM && rope.size(2) == DSV3_ROPE_DIM &&
                latent.size(0) == rope.size(0) && latent.size(1) == rope.size(1) && latent.size(0) == scale.size(0) && latent.size(1) == scale.size(1),
            "a cache is latent [pages, page_size, 512], rope [pages, page_size, 64], scale [pages, page_size]");
    if (latent.scalar_type() != at::kFloat8_e4m3fn || rope.scalar_type() != at::kBFloat16 || scale.scalar_type() != at::kFloat)
        raise(PyExc_NotImplementedError, "a cache is float8_e4m3fn latents, bfloat16 rotated values and float32 scales");
    if (latent.size(1) > (1 << 30)) raise(PyExc_NotImplementedError, "page_size is at most 2^30");
    return {latent, rope, scale,
            {latent.data_ptr(), rope.data_ptr(), static_cast<float*>(scale.data_ptr()), latent.size(0), static_cast<int>(latent.size(1)), nullptr, 0, 0, 0}};
}

const int32_t* int32_arg(const at::Tensor& t, int64_t want, const char* what) {
    require(t.dim() == 1 && t.size(0) == want && t.is_contiguous() && t.scalar_type() == at::kInt, what);
    return static_cast<const int32_t*>(t.const_data_ptr());
}

void block_table_arg(const at::Tensor& t, dsv3_latent_cache_t* c) {
    require(t.dim() == 2 && t.scalar_type() == at::kInt && (t.stride(1) == 1 || t.size(1) <= 1), "block_table must be int32 [sequences, pages]");
    if (t.size(0) > 0x7FFFFFFF) raise(PyExc_NotImplementedError, "2^31 sequences or more");
    c->pages = static_cast<const int32_t*>(t.const_data_ptr());
    c->pages_stride = t.size(0) > 1 ? t.stride(0) : 0;
    c->pages_width = t.size(1);
    c->n_seqs = static_cast<int>(t.size(0));
}

// (latent, rope, scale, kv, weight, freqs, positions, slots, eps)
PyObject* py_latent_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 9);
        const CachePlanes p = cache_arg(args[0], args[1], args[2]);
        const at::Tensor &kv = tensor_arg(args[3]), &w = tensor_arg(args[4]), &f = tensor_arg(args[5]), &pos = tensor_arg(args[6]), &slots = tensor_arg(args[7]);
        const double eps = PyFloat_AsDouble(args[8]);
        if (eps == -1.0 && PyErr_Occurred()) throw PythonError{};
        const int64_t width = DSV3_LATENT_DIM + DSV3_ROPE_DIM;
        require(kv.dim() >= 1 && kv.size(-1) == width, "kv must be [..., 576]");
        const int64_t tokens = kv.numel() / width;
        // rows of any one stride: [tokens, 576] cut from something wider, or anything contiguous
        int64_t stride = width;
        if (!kv.is_contiguous()) {
            require(kv.dim() == 2 && kv.stride(1) == 1, "kv must be contiguous, or 2-D with contiguous rows");
            stride = kv.stride(0);
        }
        require(w.dim() == 1 && w.size(0) == DSV3_LATENT_DIM && w.is_contiguous(), "the norm's weight must be a contiguous [512]");
        require(f.dim() == 2 && f.size(1) == DSV3_ROPE_DIM / 2 && f.is_contiguous() && f.scalar_type() == at::kComplexFloat,
                "freqs_cis must be a contiguous complex64 [positions, 32]");
        require(pos.numel() == tokens && slots.numel() == tokens && pos.is_contiguous() && slots.is_contiguous() && pos.scalar_type() == at::kLong &&
                    slots.scalar_type() == at::kLong,
                "positions and slots must be contiguous int64, one per token");
        const c10::Device dev = require_cuda(p.latent, p.rope, p.scale, kv, w, f, pos, slots);
        if (kv.scalar_type() != at::kBFloat16 || (w.scalar_type() != at::kBFloat16 && w.scalar_type() != at::kFloat))
            raise(PyExc_NotImplementedError, "latent_cache_write takes bfloat16 kv and a bfloat16 or float32 norm weight");
        const void *kvp = kv.const_data_ptr(), *wp = w.const_data_ptr();
        const float* fp = static_cast<const float*>(f.const_data_ptr());
        const int64_t *pp = static_cast<const int64_t*>(pos.const_data_ptr()), *sp = static_cast<const int64_t*>(slots.const_data_ptr());
        const int64_t n_pos = f.size(0);
        const int fp32 = w.scalar_type() == at::kFloat;
        call_library(dev, [&](dsv3_stream_t st) {
            return dsv3_latent_write(&p.c, kvp, stride, wp, fp32, static_cast<float>(eps), fp, n_pos, pp, sp, tokens, st);
        });
        Py_RETURN_NONE;
    });
}

// (latent, rope, scale, block_table, cu_seqlens, total) -> (latent, rope)
PyObject* py_latent_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 6);
        CachePlanes p = cache_arg(args[0], args[1], args[2]);
        const at::Tensor &table = tensor_arg(args[3]), &cu = tensor_arg(args[4]);
        block_table_arg(table, &p.c);
        const int32_t* cup = int32_arg(cu, table.size(0) + 1, "cu_seqlens must be contiguous int32 [sequences + 1]");
        const int64_t total = int_arg(args[5]);
        require(total >= 0, "total must not be negative");
        const c10::Device dev = require_cuda(p.latent, p.rope, p.scale, table, cu);
        at::Tensor latent = new_cuda({total, DSV3_LATENT_DIM}, at::kBFloat16, dev), rope = new_cuda({total, DSV3_ROPE_DIM}, at::kBFloat16, dev);
        void *lp = latent.data_ptr(), *rp = rope.data_ptr();
        call_library(dev, [&](dsv3_stream_t st) { return dsv3_latent_read(&p.c, cup, total, lp, rp, st); });
        return wrap_pair(std::move(latent), std::move(rope));
    });
}

// (latent, rope, scale, block_table, first, path, count)
PyObject* py_latent_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 7);
        CachePlanes p = cache_arg(args[0], args[1], args[2]);
        const at::Tensor &table = tensor_arg(args[3]), &first = tensor_arg(args[4]), &path = tensor_arg(args[5]), &count = tensor_arg(args[6]);
        block_table_arg(table, &p.c);
        const int32_t* fp = int32_arg(first, table.size(0), "first must be contiguous int32 [sequences]");
        const int32_t* cp = int32_arg(count, table.size(0), "count must be contiguous int32 [sequences]");
        require(path.dim() == 2 && path.size(0) == table.size(0) && path.scalar_type() == at::kInt && (path.stride(1) == 1 || path.size(1) <= 1),
                "path must be int32 [sequences, drafts]");
        if (path.size(1) > 0x7FFFFFFF) raise(PyExc_NotImplementedError, "2^31 drafts or more");
        const c10::Device dev = require_cuda(p.latent, p.rope, p.scale, table, first, path, count);
        const int32_t* pp = static_cast<const int32_t*>(path.const_data_ptr());
        const int64_t stride = path.size(0) > 1 ? path.stride(0) : 0;
        const int drafts = static_cast<int>(path.size(1));
        call_library(dev, [&](dsv3_stream_t st) { return dsv3_latent_keep(&p.c, fp, pp, stride, drafts, cp, st); });
        Py_RETURN_NONE;
    });
}

// Query rows [tokens, heads, width], or [batch, tokens, heads, width] with batch and tokens one stride apart.
struct QueryRows {
    int64_t tokens, heads, token_stride, head_stride;
};
QueryRows query_rows(const at::Tensor& q, int64_t width) {
    require((q.dim() == 3 || q.dim() == 4) && q.size(-1) == width, "queries must be [tokens, heads, 512] and [tokens, heads, 64], or with a batch in front");
    require(q.stride(-1) == 1, "the last dimension of the queries must be contiguous");
    QueryRows r{q.size(-3), q.size(-2), q.stride(-3), q.size(-2) > 1 ? q.stride(-2) : 0};
    if (q.dim() == 4) {
        require(q.size(0) <= 1 || q.size(1) <= 1 || q.stride(0) == q.size(1) * q.stride(1), "batch and tokens of the queries must have one stride");
        if (q.size(1) <= 1) r.token_stride = q.stride(0);
        r.tokens *= q.size(0);
    }
    if (r.tokens <= 1) r.token_stride = 0;
    return r;
}

// (q_latent, q_rope, latent, rope, scale, block_table, seq_lens, softmax_scale, cu_seqlens_q or None, tree_mask or None, return_lse) -> out, or (out, lse)
PyObject* py_latent_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 11);
        const at::Tensor &ql = tensor_arg(args[0]), &qr = tensor_arg(args[1]);
        CachePlanes p = cache_arg(args[2], args[3], args[4]);
        const at::Tensor &table = tensor_arg(args[5]), &lens = tensor_arg(args[6]);
        const double scale = PyFloat_AsDouble(args[7]);
        if (scale == -1.0 && PyErr_Occurred()) throw PythonError{};
        const int with_lse = PyObject_IsTrue(args[10]);
        if (with_lse < 0) throw PythonError{};
        block_table_arg(table, &p.c);
        const QueryRows l = query_rows(ql, DSV3_LATENT_DIM), r = query_rows(qr, DSV3_ROPE_DIM);
        require(l.tokens == r.tokens && l.heads == r.heads && ql.dim() == qr.dim(), "q_latent and q_rope must have the same tokens and heads");
        const int32_t* lp = int32_arg(lens, table.size(0), "seq_lens must be contiguous int32 [sequences]");
        const c10::Device dev = require_cuda(ql, qr, p.latent, p.rope, p.scale, table, lens);
        if (ql.scalar_type() != at::kBFloat16 || qr.scalar_type() != at::kBFloat16)
            raise(PyExc_NotImplementedError, "latent_attention takes bfloat16 queries");
        const int32_t* cup = nullptr;
        if (args[8] != Py_None) {
            const at::Tensor& cu = tensor_arg(args[8]);
            require_cuda(ql, cu);
            cup = int32_arg(cu, table.size(0) + 1, "cu_seqlens_q must be contiguous int32 [sequences + 1]");
        } else {
            require(l.tokens == 0 || (table.size(0) > 0 && l.tokens % table.size(0) == 0 && (ql.dim() == 3 || ql.size(0) == table.size(0))),
                    "without cu_seqlens_q every sequence has the same number of queries");
        }
        const int64_t* tp = nullptr;
        if (args[9] != Py_None) {
            const at::Tensor& tree = tensor_arg(args[9]);
            require_cuda(ql, tree);
            require(tree.numel() == l.tokens && tree.is_contiguous() && tree.scalar_type() == at::kLong, "tree_mask must be contiguous int64, a word per query");
            tp = static_cast<const int64_t*>(tree.const_data_ptr());
        }
        if (l.heads > 1024) raise(PyExc_NotImplementedError, "latent_attention takes at most 1024 heads");
        c10::SmallVector<int64_t, 4> sizes(ql.sizes().begin(), ql.sizes().end());
        at::Tensor out = new_cuda(sizes, at::kBFloat16, dev), lse;
        sizes.pop_back();
        if (with_lse) lse = new_cuda(sizes, at::kFloat, dev);
        c10::cuda::OptionalCUDAGuard guard;                                    // (the size is that of the current device)
        if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
        const size_t need = dsv3_latent_attention_workspace_bytes(l.tokens, static_cast<int>(l.heads), p.c.n_seqs, p.c.pages_width * p.c.page_size);
        // (given back after the launches: torch hands the memory out again in the stream's order)
        const at::Tensor ws = need ? new_cuda({static_cast<int64_t>(need)}, at::kByte, dev) : at::Tensor();
        void *op = out.data_ptr(), *wp = need ? ws.data_ptr() : nullptr;
        float* sp = with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
        const void *qlp = ql.const_data_ptr(), *qrp = qr.const_data_ptr();
        call_library(dev, [&](dsv3_stream_t st) {
            return dsv3_latent_attention(&p.c, qlp, l.token_stride, l.head_stride, qrp, r.token_stride, r.head_stride, l.tokens, static_cast<int>(l.heads), lp,
                                         cup, tp, static_cast<float>(scale), op, sp, wp, need, st);
        });
        return with_lse ? wrap_pair(std::move(out), std::move(lse)) : wrap(std::move(out));
    });
}
