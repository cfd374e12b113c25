// ------------------------------------------------------------------ attention over expanded keys and values, rotary positions (part of host.cpp)
// [tokens, heads, width], or [batch, tokens, heads, width] with batch and tokens one stride apart.
struct HeadRows {
    int64_t batch, tokens, heads, token_stride, head_stride;      // tokens: of the whole batch
};
HeadRows head_rows(const at::Tensor& t, int64_t width, const char* shape) {
    require((t.dim() == 3 || t.dim() == 4) && (width < 0 || t.size(-1) == width), shape);
    require(t.stride(-1) == 1 || t.size(-1) <= 1, "the last dimension of heads must be contiguous");
    HeadRows r{t.dim() == 4 ? t.size(0) : -1, t.size(-3), t.size(-2), t.stride(-3), t.size(-2) > 1 ? t.stride(-2) : 0};
    if (t.dim() == 4) {
        require(t.size(0) <= 1 || t.size(1) <= 1 || t.stride(0) == t.size(1) * t.stride(1), "batch and tokens must have one stride");
        if (t.size(1) <= 1) r.token_stride = t.stride(0);
        r.tokens *= t.size(0);
    }
    if (r.tokens <= 1) r.token_stride = 0;
    return r;
}

const int32_t* offsets_arg(PyObject* o, const at::Tensor& beside, int64_t* n_seqs) {
    if (o == Py_None) return nullptr;
    const at::Tensor& t = tensor_arg(o);
    require_cuda(beside, t);
    require(t.dim() == 1 && t.size(0) >= 1 && t.is_contiguous() && t.scalar_type() == at::kInt, "cu_seqlens must be contiguous int32 [sequences + 1]");
    require(*n_seqs < 0 || *n_seqs == t.size(0) - 1, "cu_seqlens_q and cu_seqlens_k must be of the same sequences");
    *n_seqs = t.size(0) - 1;
    return static_cast<const int32_t*>(t.const_data_ptr());
}

// (q_nope, q_rope, k_nope, k_rope, v, softmax_scale, cu_seqlens_q or None, cu_seqlens_k or None, causal, return_lse) -> out, or (out, lse)
PyObject* py_expanded_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 10);
        const at::Tensor &qn = tensor_arg(args[0]), &qr = tensor_arg(args[1]), &kn = tensor_arg(args[2]), &kr = tensor_arg(args[3]), &v = tensor_arg(args[4]);
        const double scale = PyFloat_AsDouble(args[5]);
        if (scale == -1.0 && PyErr_Occurred()) throw PythonError{};
        const int causal = PyObject_IsTrue(args[8]), with_lse = PyObject_IsTrue(args[9]);
        if (causal < 0 || with_lse < 0) throw PythonError{};
        const HeadRows q = head_rows(qn, DSV3_NOPE_DIM, "q_nope must be [tokens, heads, 128], or with a batch in front"),
                       r = head_rows(qr, DSV3_ROPE_DIM, "q_rope must be [tokens, heads, 64], or with a batch in front"),
                       k = head_rows(kn, DSV3_NOPE_DIM, "k_nope must be [tokens, heads, 128], or with a batch in front"),
                       x = head_rows(v, DSV3_VALUE_DIM, "v must be [tokens, heads, 128], or with a batch in front");
        require(q.tokens == r.tokens && q.heads == r.heads && q.batch == r.batch, "q_nope and q_rope must have the same tokens and heads");
        require(k.tokens == x.tokens && k.heads == x.heads && k.batch == x.batch && k.heads == q.heads, "k_nope and v must have the same tokens, and the heads of the queries");
        // the rotated part of the keys: no heads
        require(kr.dim() == kn.dim() - 1 && kr.size(-1) == DSV3_ROPE_DIM && kr.size(-2) == kn.size(-3) && (kr.dim() == 2 || kr.size(0) == kn.size(0)),
                "k_rope must be [tokens, 64], or with a batch in front, and have the tokens of k_nope");
        require(kr.stride(-1) == 1, "the last dimension of k_rope must be contiguous");
        int64_t kr_stride = kr.stride(-2);
        if (kr.dim() == 3) {
            require(kr.size(0) <= 1 || kr.size(1) <= 1 || kr.stride(0) == kr.size(1) * kr.stride(1), "batch and tokens must have one stride");
            if (kr.size(1) <= 1) kr_stride = kr.stride(0);
        }
        if (k.tokens <= 1) kr_stride = 0;
        const c10::Device dev = require_cuda(qn, qr, kn, kr, v);
        for (const at::Tensor* t : {&qn, &qr, &kn, &kr, &v})
            if (t->scalar_type() != at::kBFloat16) raise(PyExc_NotImplementedError, "expanded_attention takes bfloat16 queries, keys and values");
        int64_t n_seqs = -1;
        const int32_t *cu_q = offsets_arg(args[6], qn, &n_seqs), *cu_k = offsets_arg(args[7], qn, &n_seqs);
        if (!cu_q) {
            require(n_seqs < 0 || n_seqs == std::max<int64_t>(q.batch, 1), "without cu_seqlens_q the queries' batch must be the sequences");
            n_seqs = std::max<int64_t>(q.batch, q.batch < 0 ? 1 : 0);
        }
        if (!cu_k) require(n_seqs == (k.batch < 0 ? 1 : k.batch), "without cu_seqlens_k the keys' batch must be the sequences");
        if (n_seqs > 0x7FFFFFFF) raise(PyExc_NotImplementedError, "2^31 sequences or more");
        if (q.heads > 1024) raise(PyExc_NotImplementedError, "expanded_attention takes at most 1024 heads");
        if (!(scale > 0.0) || scale > 1e30) raise(PyExc_ValueError, "softmax_scale must be positive and finite");
        c10::SmallVector<int64_t, 4> sizes(qn.sizes().begin(), qn.sizes().end());
        sizes.back() = DSV3_VALUE_DIM;
        at::Tensor out = new_cuda(sizes, at::kBFloat16, dev), lse;
        sizes.pop_back();
        if (with_lse) lse = new_cuda(sizes, at::kFloat, dev);
        c10::cuda::OptionalCUDAGuard guard;                                    // (the size is that of the current device)
        if (dev.index() != c10::cuda::current_device()) guard.set_device(dev);
        const size_t need = dsv3_expanded_attention_workspace_bytes(q.tokens, k.tokens, static_cast<int>(q.heads), static_cast<int>(n_seqs), cu_q != nullptr, causal);
        // (given back after the launches: torch hands the memory out again in the stream's order)
        const at::Tensor ws = need ? new_cuda({static_cast<int64_t>(need)}, at::kByte, dev) : at::Tensor();
        const dsv3_expanded_attention_t a = {qn.const_data_ptr(), q.token_stride, q.head_stride, qr.const_data_ptr(), r.token_stride, r.head_stride,
                                             kn.const_data_ptr(), k.token_stride, k.head_stride, kr.const_data_ptr(), kr_stride,
                                             v.const_data_ptr(), x.token_stride, x.head_stride, q.tokens, k.tokens, static_cast<int>(q.heads),
                                             static_cast<int>(n_seqs), cu_q, cu_k, causal, static_cast<float>(scale), out.data_ptr(),
                                             with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr};
        void* const wp = need ? ws.data_ptr() : nullptr;
        if (q.tokens > 0 && n_seqs > 0) call_library(dev, [&](dsv3_stream_t st) { return dsv3_expanded_attention(&a, wp, need, st); });
        return with_lse ? wrap_pair(std::move(out), std::move(lse)) : wrap(std::move(out));
    });
}

// (outs, lses, return_lse) -> out, or (out, lse)
PyObject* py_attention_join(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 3);
        const int with_lse = PyObject_IsTrue(args[2]);
        if (with_lse < 0) throw PythonError{};
        require(PyTuple_Check(args[0]) && PyTuple_Check(args[1]), "outs and lses must be sequences");
        const Py_ssize_t parts = PyTuple_GET_SIZE(args[0]);
        require(parts >= 1 && PyTuple_GET_SIZE(args[1]) == parts, "there must be a part, and an lse to each");
        if (parts > 32) raise(PyExc_NotImplementedError, "attention_join takes at most 32 parts");
        const void* outs[32];
        const float* lses[32];
        const at::Tensor& first = tensor_arg(PyTuple_GET_ITEM(args[0], 0));
        require(first.dim() >= 1, "parts must be [..., dim]");
        const c10::Device dev = require_cuda(first);
        for (Py_ssize_t i = 0; i < parts; ++i) {
            const at::Tensor &o = tensor_arg(PyTuple_GET_ITEM(args[0], i)), &l = tensor_arg(PyTuple_GET_ITEM(args[1], i));
            require_cuda(first, o, l);
            require(o.sizes() == first.sizes() && l.sizes() == first.sizes().slice(0, first.dim() - 1), "parts must have one shape [..., dim], and their lses [...]");
            require(o.is_contiguous() && l.is_contiguous(), "parts and their lses must be contiguous");
            if (o.scalar_type() != at::kBFloat16 || l.scalar_type() != at::kFloat) raise(PyExc_NotImplementedError, "attention_join takes bfloat16 parts and float32 lses");
            outs[i] = o.const_data_ptr(), lses[i] = static_cast<const float*>(l.const_data_ptr());
        }
        const int64_t dim = first.size(-1), rows = dim > 0 ? first.numel() / dim : 0, l_rows = tensor_arg(PyTuple_GET_ITEM(args[1], 0)).numel();
        if (dim > 2048) raise(PyExc_NotImplementedError, "attention_join takes at most 2048 values a row");
        if (dim == 0 && with_lse && l_rows > 0) raise(PyExc_NotImplementedError, "attention_join does not join the logarithms of rows without values");
        c10::SmallVector<int64_t, 6> sizes(first.sizes().begin(), first.sizes().end());
        at::Tensor out = new_cuda(sizes, at::kBFloat16, dev), lse;
        sizes.pop_back();
        if (with_lse) lse = new_cuda(sizes, at::kFloat, dev);
        void* const op = out.data_ptr();
        float* const lp = with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
        if (rows > 0)
            call_library(dev, [&](dsv3_stream_t st) { return dsv3_attention_join(outs, lses, static_cast<int>(parts), rows, static_cast<int>(dim), op, lp, st); });
        return with_lse ? wrap_pair(std::move(out), std::move(lse)) : wrap(std::move(out));
    });
}

double double_arg(PyObject* o) {
    const double d = PyFloat_AsDouble(o);
    if (d == -1.0 && PyErr_Occurred()) throw PythonError{};
    return d;
}

// (length, dim, theta, factor, original_length, beta_fast, beta_slow, start, device index or None) -> complex64 [length, dim / 2]
PyObject* py_rotary_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 9);
        const int64_t length = int_arg(args[0]), dim = int_arg(args[1]), original = int_arg(args[4]), start = int_arg(args[7]);
        const double theta = double_arg(args[2]), factor = double_arg(args[3]), fast = double_arg(args[5]), slow = double_arg(args[6]);
        if (length < 0 || start < 0) raise(PyExc_ValueError, "length and start must not be negative");
        if (dim < 2 || dim % 2 != 0 || dim > 256) raise(PyExc_ValueError, "dim must be even, from 2 to 256");
        const c10::Device dev(c10::kCUDA, static_cast<c10::DeviceIndex>(args[8] == Py_None ? c10::cuda::current_device() : int_arg(args[8])));
        at::Tensor out = new_cuda({length, dim / 2}, at::kComplexFloat, dev);
        float* const op = static_cast<float*>(out.data_ptr());
        call_library(dev, [&](dsv3_stream_t st) { return dsv3_rotary_table(static_cast<int>(dim), theta, factor, original, fast, slow, start, length, op, st); });
        return wrap(std::move(out));
    });
}

// Bytes between a tensor's first and behind its last element.
std::pair<const char*, const char*> extent(const at::Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    const char* const p = static_cast<const char*>(t.const_data_ptr());
    return {p, p + (last + 1) * static_cast<int64_t>(t.element_size())};
}

// (x, freqs) -> whether rotary takes a batch [batch, tokens, heads, dim] as it lies, with the angles [tokens, dim / 2] of all of its heads' values: tokens one stride apart, rows at multiples of 16 bytes
PyObject* py_rotary_takes(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 2);
        const at::Tensor &x = tensor_arg(args[0]), &f = tensor_arg(args[1]);
        if (x.dim() != 4) raise(PyExc_ValueError, "x must be [batch, tokens, heads, dim]");
        const int64_t batch = x.size(0), tokens = x.size(1), each = 16 / std::max<int64_t>(1, static_cast<int64_t>(x.element_size())), step = tokens > 1 ? x.stride(1) : x.stride(0);
        return PyBool_FromLong(f.dim() == 2 && f.size(0) == tokens && f.size(1) == x.size(3) / 2 && f.is_contiguous() && x.stride(3) == 1 &&
                               (batch <= 1 || tokens <= 1 || x.stride(0) == tokens * step) && (batch * tokens <= 1 || step % each == 0) && (x.size(2) <= 1 || x.stride(2) % each == 0) &&
                               reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0);
    });
}

// (x, freqs, positions or None, half_layout, offset, inverse, out or None) -> out, or None where autograd is to have a gradient, which is the caller's part
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
    return guarded([&]() -> PyObject* {
        want_args(n, 7);
        const at::Tensor &x = tensor_arg(args[0]), &f = tensor_arg(args[1]);
        if (c10::GradMode::is_enabled() && (x.requires_grad() || f.requires_grad() || (args[6] != Py_None && tensor_arg(args[6]).requires_grad()))) Py_RETURN_NONE;
        const int half = PyObject_IsTrue(args[3]), inverse = PyObject_IsTrue(args[5]);
        if (half < 0 || inverse < 0) throw PythonError{};
        const int64_t offset = int_arg(args[4]);
        const HeadRows r = head_rows(x, -1, "x must be [tokens, heads, dim], or with a batch in front");
        require(f.dim() == 2 && f.is_contiguous() && f.scalar_type() == at::kComplexFloat, "freqs_cis must be a contiguous complex64 [positions, rotated / 2]");
        const int64_t dim = x.size(-1), rotated = 2 * f.size(1), per = x.size(-3);
        require(offset >= 0 && offset + rotated <= dim, "the rotated part must lie within a head");
        const c10::Device dev = require_cuda(x, f);
        const int dtype = x.scalar_type() == at::kBFloat16 ? DSV3_BF16 : x.scalar_type() == at::kHalf ? DSV3_FP16 : x.scalar_type() == at::kFloat ? DSV3_FP32 : -1;
        if (dtype < 0) raise(PyExc_NotImplementedError, "rotary takes bfloat16, float16 or float32");
        if (dim > 1024 || r.heads > 0x7FFFFFFF) raise(PyExc_NotImplementedError, "rotary takes heads of at most 1024 values");
        const int64_t* pp = nullptr;
        if (args[2] != Py_None) {
            const at::Tensor& p = tensor_arg(args[2]);
            require_cuda(x, p);
            require(p.numel() == r.tokens && p.is_contiguous() && p.scalar_type() == at::kLong, "positions must be contiguous int64, one per token");
            pp = static_cast<const int64_t*>(p.const_data_ptr());
        } else {
            require(f.size(0) >= per, "without positions freqs_cis must have a row for every token of a sequence");
        }
        at::Tensor out;
        HeadRows o;
        if (args[6] == Py_None) {
            out = new_cuda(x.sizes(), x.scalar_type(), dev);
            o = head_rows(out, -1, "out");
        } else {
            out = tensor_arg(args[6]);
            require_cuda(x, out);
            require(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type(), "out must have x's shape and type");
            o = head_rows(out, -1, "out must be [tokens, heads, dim], or with a batch in front");
            require(o.heads <= 1 || o.head_stride != 0, "out must not hold several heads in one place");
            require(o.tokens <= 1 || o.token_stride != 0, "out must not hold several tokens in one place");
            if (out.numel() > 0 && out.const_data_ptr() != x.const_data_ptr()) {
                const auto a = extent(x), b = extent(out);
                require(a.second <= b.first || b.second <= a.first, "out must be x itself, or not overlap it");
            }
        }
        const void* const xp = x.const_data_ptr();
        const float* const fp = static_cast<const float*>(f.const_data_ptr());
        void* const op = out.data_ptr();
        const int64_t positions = f.size(0);
        if (x.numel() > 0)
            call_library(dev, [&](dsv3_stream_t st) {
                return dsv3_rotary(xp, r.token_stride, r.head_stride, op, o.token_stride, o.head_stride, dtype, r.tokens, static_cast<int>(r.heads), static_cast<int>(dim), fp,
                                   positions, pp, std::max<int64_t>(per, 1), static_cast<int>(offset), static_cast<int>(rotated), half, inverse, st);
            });
        return wrap(std::move(out));
    });
}
