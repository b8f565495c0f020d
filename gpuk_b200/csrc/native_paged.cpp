// The CPython functions of the paged KV cache (module `gpuk_b200._native`, see native.cpp): arguments checked, results and workspaces allocated on the current stream of the tensors'
// device, errors raised.  There are no operators to hand a call back to, so what cannot be taken is refused.
#include "native.hpp"

#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace gpuk_native {
namespace {

// To a trace the call would not be there: its result would be a constant and nothing be written on replay.  Function modes are not asked: most only say on which device new tensors are made.
void expect_unwatched(const char *what) {
    TORCH_CHECK(!watched(), "gpuk::", what, " is no operator that a dispatch mode, a trace or a functional transform could see: call it outside of them");
}
// A dense CUDA tensor on the given device (-1: any) that no transform or gradient has an interest in.
const Tensor &paged_arg(PyObject *o, const char *what, int device) {
    const Tensor &t = tensor_arg(o, what);
    TORCH_CHECK(plain_class(o) && t.layout() == at::kStrided, "gpuk: ", what, " must be a plain tensor");
    TORCH_CHECK(t.is_cuda(), "gpuk: ", what, " must be a CUDA tensor");
    TORCH_CHECK(device < 0 || t.get_device() == device, "gpuk: ", what, " is on another device");
    if (t.unsafeGetTensorImpl()->autograd_meta()) {      // few tensors have any
        TORCH_CHECK(!(t.requires_grad() && c10::GradMode::is_enabled()), "gpuk: ", what, " requires a gradient, and the paged cache's calls have none: call them under torch.no_grad()");
        TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), "gpuk: ", what, " has a forward-mode tangent, which the paged cache's calls would drop");
    }
    return t;
}
const Tensor &ints_arg(PyObject *o, const char *what, int device, at::ScalarType type, int64_t count) {
    const Tensor &t = paged_arg(o, what, device);
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.is_contiguous(), "gpuk: ", what, " must be a contiguous one-dimensional tensor of ", type);
    TORCH_CHECK(t.size(0) == count, "gpuk: ", what, " has ", t.size(0), " elements, needs ", count);
    return t;
}
// A matrix of int32 whose rows are contiguous.
const Tensor &rows_arg(PyObject *o, const char *what, int device, int64_t rows) {
    const Tensor &t = paged_arg(o, what, device);
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), "gpuk: ", what, " must be a two-dimensional int32 tensor with contiguous rows");
    TORCH_CHECK(t.size(0) == rows, "gpuk: ", what, " has ", t.size(0), " rows, needs ", rows);
    return t;
}
int dtype_of(const Tensor &t, const char *what) {
    TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "gpuk: ", what, " must be bfloat16 or float16");
    return t.scalar_type() == at::kBFloat16 ? GPUK_DTYPE_BF16 : GPUK_DTYPE_F16;
}
// The stride of a dimension; one that is never stepped along gets one that the kernels take.
int64_t stride_of(const Tensor &t, int dim) { return t.size(dim) <= 1 ? std::max<int64_t>(8, (t.size(-1) + 7) / 8 * 8) : t.stride(dim); }
// [tokens, heads, head_dim] with contiguous heads.
const Tensor &heads_arg(PyObject *o, const char *what, int device) {
    const Tensor &t = paged_arg(o, what, device);
    TORCH_CHECK(t.dim() == 3 && (t.size(2) <= 1 || t.stride(2) == 1), "gpuk: ", what, " must be [tokens, heads, head_dim] with contiguous heads");
    dtype_of(t, what);
    return t;
}
// Whether two views with the same strides share an element: whether `distance` is a sum of steps along the dimensions, the longest first, each of which is longer than all shorter ones together.
struct Step {
    int64_t stride, least, most;
};
bool meet(int64_t distance, const Step *steps, int n) {
    if (n == 0) return distance == 0;
    int64_t c = distance / steps->stride;
    if (c * steps->stride > distance) --c;
    for (int i = 0; i < 2; ++i, ++c)
        if (c >= steps->least && c <= steps->most && meet(distance - c * steps->stride, steps + 1, n - 1)) return true;
    return false;
}
// Whether two tensors may share an element: exactly for views of the same strides (heads of one projection's output, keys and values in one allocation), by the bytes that they span for others.
bool overlap(const Tensor &a, const Tensor &b) {
    if (!a.numel() || !b.numel()) return false;
    auto end = [](const Tensor &t) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        return static_cast<const char *>(t.const_data_ptr()) + (last + 1) * t.element_size();
    };
    const char *const at = static_cast<const char *>(a.const_data_ptr()), *const bt = static_cast<const char *>(b.const_data_ptr());
    if (at >= end(b) || bt >= end(a)) return false;
    const int64_t size = a.element_size();
    if (a.dim() != b.dim() || a.dim() > 5 || size != static_cast<int64_t>(b.element_size()) || (bt - at) % size) return true;
    Step steps[5];
    int n = 0;
    for (int64_t d = 0; d < a.dim(); ++d) {
        const int64_t na = a.size(d), nb = b.size(d), stride = na > 1 ? a.stride(d) : b.stride(d);
        if (na <= 1 && nb <= 1) continue;
        if (stride <= 0 || (na > 1 && nb > 1 && b.stride(d) != stride)) return true;
        steps[n++] = {stride, 1 - nb, na - 1};
    }
    std::sort(steps, steps + n, [](const Step &x, const Step &y) { return x.stride > y.stride; });
    int64_t shorter = 0;
    for (int i = n - 1; i >= 0; --i) {
        if (shorter >= steps[i].stride) return true;
        shorter += std::max(steps[i].most, -steps[i].least) * steps[i].stride;
    }
    return meet((bt - at) / size, steps, n);
}
bool same_place(const Tensor &a, const Tensor &b) { return a.const_data_ptr() == b.const_data_ptr() && a.strides() == b.strides(); }

// k_pages and v_pages [pages, kv_heads, page_size, head_dim], or with a dimension of layers in front.
struct Pages {
    const Tensor &k, &v;
    gpuk_pages c = {};
    int64_t layers = 1, layer_stride = 0;
    Pages(PyObject *ko, PyObject *vo, int device, bool layered, bool written) : k(paged_arg(ko, "k_pages", device)), v(paged_arg(vo, "v_pages", k.get_device())) {
        const int at = layered && k.dim() == 5 ? 1 : 0;
        TORCH_CHECK(k.dim() == 4 + at && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "gpuk: k_pages and v_pages must be [pages, kv_heads, page_size, head_dim], ",
                    "of one size and type");
        c.dtype = dtype_of(k, "k_pages");
        for (int d = 0; d < k.dim(); ++d) TORCH_CHECK(stride_of(k, d) == stride_of(v, d), "gpuk: k_pages and v_pages must have the same strides");
        TORCH_CHECK(k.size(3 + at) <= 1 || k.stride(3 + at) == 1, "gpuk: a token's head must be contiguous in k_pages and v_pages");
        if (written) {
            for (int d = 0; d < k.dim(); ++d) TORCH_CHECK(k.size(d) <= 1 || k.stride(d) > 0, "gpuk: k_pages and v_pages repeat their elements");
            TORCH_CHECK(!overlap(k, v), "gpuk: k_pages and v_pages overlap");
        }
        if (at) layers = k.size(0), layer_stride = stride_of(k, 0);
        c.k = k.data_ptr(), c.v = v.data_ptr();
        c.page_stride = stride_of(k, at), c.head_stride = stride_of(k, 1 + at), c.row_stride = stride_of(k, 2 + at);
        c.num_pages = k.size(at), c.kv_heads = int_size(k.size(1 + at)), c.page_size = int_size(k.size(2 + at)), c.head_dim = int_size(k.size(3 + at));
    }
};
double float_arg(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
PyObject *wrap_or_none(Tensor t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(t));
}
// A given result, or a new one.
Tensor heads_out(PyObject *o, const Tensor &like, const char *what) {
    if (o == Py_None) return empty_like_on(like, like.sizes(), like.scalar_type());
    const Tensor &t = heads_arg(o, what, like.get_device());
    TORCH_CHECK(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type(), "gpuk: ", what, " has another size or type");
    // a token's heads behind one another, or a head's tokens
    const int64_t n = t.size(2), tokens = t.size(0), heads = t.size(1), token = tokens > 1 ? t.stride(0) : n * heads, head = heads > 1 ? t.stride(1) : n;
    TORCH_CHECK(!t.numel() || (head >= n && token >= (tokens > 1 ? n : 0) && (heads <= 1 || tokens <= 1 || token >= heads * head || head >= tokens * token)), "gpuk: ", what,
                " repeats its elements");
    return t;
}

// Contiguous tensors of several sizes and types from one allocation: a call to the allocator for each is what a plan would cost the host most.
class Pool {
    int64_t bytes_ = 0;
    c10::Storage storage_;

  public:
    int64_t add(int64_t elements, int64_t element_size) {
        const int64_t at = bytes_;
        bytes_ += (elements * element_size + 15) / 16 * 16;
        return at / element_size;      // 16 is a multiple of it
    }
    void allocate(const Tensor &like) { storage_ = empty_like_on(like, {std::max<int64_t>(bytes_, 1)}, at::kByte).storage(); }
    Tensor take(int64_t offset, at::IntArrayRef sizes, at::ScalarType type) const {
        Tensor t = at::detail::make_tensor<at::TensorImpl>(c10::Storage(storage_), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
        t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
        t.unsafeGetTensorImpl()->set_storage_offset(offset);
        return t;
    }
};

}  // namespace

// paged_plan(lens, new_lens, tables, held, free, free_count, page_size, total, parents or None, max_new, held_out or None, free_count_out or None)
//   -> (starts, positions, slots, masks or None, held, free_count)
PyObject *paged_plan(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect_args(n, 12, "paged_plan");
    expect_unwatched("paged_plan");
    const Tensor &lens = paged_arg(args[0], "lens", -1);
    const int dev = lens.get_device();
    TORCH_CHECK(lens.dim() == 1, "gpuk: lens must be one-dimensional");
    const int64_t batch = lens.size(0), page = int_arg(args[6]), total = int_arg(args[7]), max_new = int_arg(args[9]);
    ints_arg(args[0], "lens", dev, at::kInt, batch);
    const Tensor &fresh = ints_arg(args[1], "new_lens", dev, at::kInt, batch), &tables = rows_arg(args[2], "tables", dev, batch), &held = ints_arg(args[3], "held", dev, at::kInt, batch);
    const Tensor &free = paged_arg(args[4], "free", dev);
    ints_arg(args[4], "free", dev, at::kInt, free.numel());
    const Tensor &count = ints_arg(args[5], "free_count", dev, at::kInt, 2);
    TORCH_CHECK(batch <= 1 || tables.stride(0) >= tables.size(1), "gpuk: rows of tables overlap");
    const bool tree = args[8] != Py_None;
    int words = 0;
    const Tensor *parents = nullptr;
    if (tree) {
        parents = &ints_arg(args[8], "parents", dev, at::kInt, total);
        TORCH_CHECK(max_new >= 1 && max_new <= 256, "gpuk: paged_plan with parents needs max_new, the most new tokens of a request, from 1 to 256");
        words = static_cast<int>((max_new + 31) / 32);
    }
    Tensor held_out, count_out, starts, positions, slots, masks;
    if (args[10] != Py_None) held_out = ints_arg(args[10], "held_out", dev, at::kInt, batch);
    if (args[11] != Py_None) count_out = ints_arg(args[11], "free_count_out", dev, at::kInt, 2);
    // what is written may stand where it was read, but nowhere else among the arguments
    for (const Tensor *w : {&held_out, &count_out}) {
        if (!w->defined()) continue;
        for (const Tensor *r : {&lens, &fresh, &tables, &held, &free, &count, parents}) {
            const bool own_place = (w == &held_out && r == &held) || (w == &count_out && r == &count);
            TORCH_CHECK(!r || !overlap(*w, *r) || (own_place && same_place(*w, *r)), "gpuk: paged_plan results overlap its arguments");
        }
    }
    TORCH_CHECK(!(held_out.defined() && count_out.defined() && overlap(held_out, count_out)), "gpuk: paged_plan results overlap each other");
    for (const Tensor *w : {&tables, &free})
        for (const Tensor *r : {&lens, &fresh, &tables, &held, &free, &count, parents})
            TORCH_CHECK(!r || r == w || !overlap(*w, *r), "gpuk: paged_plan arguments overlap its tables or its list");
    {
        NoGil unlocked;
        c10::cuda::CUDAGuard guard(lens.device());
        const int rows = int_size(total);
        Pool pool;
        const int64_t at_positions = pool.add(total, 8), at_slots = pool.add(total, 8), at_masks = pool.add(total * words, 4), at_starts = pool.add(batch + 1, 4),
                      at_held = pool.add(batch, 4), at_count = pool.add(2, 4);
        pool.allocate(lens);
        if (!held_out.defined()) held_out = pool.take(at_held, {batch}, at::kInt);
        if (!count_out.defined()) count_out = pool.take(at_count, {2}, at::kInt);
        starts = pool.take(at_starts, {batch + 1}, at::kInt);
        positions = pool.take(at_positions, {total}, at::kLong), slots = pool.take(at_slots, {total}, at::kLong);
        if (tree) masks = pool.take(at_masks, {total, words}, at::kInt);
        check(gpuk_paged_plan(lens.data_ptr<int>(), fresh.data_ptr<int>(), tables.data_ptr<int>(), tables.size(0) > 1 ? tables.stride(0) : tables.size(1), int_size(tables.size(1)),
                              held.data_ptr<int>(), free.data_ptr<int>(), int_size(free.numel()), count.data_ptr<int>(), tree ? parents->data_ptr<int>() : nullptr, int_size(batch), rows,
                              int_size(page), words, starts.data_ptr<int>(), positions.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), tree ? masks.data_ptr<int>() : nullptr,
                              held_out.data_ptr<int>(), count_out.data_ptr<int>(), stream_of(lens)), "paged_plan");
    }
    PyObject *result = PyTuple_New(6);
    if (!result) throw python_error();
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(starts)));
    PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(positions)));
    PyTuple_SET_ITEM(result, 2, THPVariable_Wrap(std::move(slots)));
    PyTuple_SET_ITEM(result, 3, wrap_or_none(std::move(masks)));
    PyTuple_SET_ITEM(result, 4, THPVariable_Wrap(std::move(held_out)));
    PyTuple_SET_ITEM(result, 5, THPVariable_Wrap(std::move(count_out)));
    return result;
    END_HANDLE_TH_ERRORS
}

// rope(x [tokens, heads, head_dim], positions, turns, amplitude, layout, out or None) -> out
PyObject *rope(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect_args(n, 6, "rope");
    expect_unwatched("rope");
    const Tensor &x = heads_arg(args[0], "x", -1);
    const int dev = x.get_device();
    const Tensor &pos = ints_arg(args[1], "positions", dev, at::kLong, x.size(0)), &turns = paged_arg(args[2], "frequencies", dev);
    ints_arg(args[2], "frequencies", dev, at::kLong, turns.numel());
    const double amplitude = float_arg(args[3]);
    const int64_t layout = int_arg(args[4]);
    Tensor out;
    {
        NoGil unlocked;
        c10::cuda::CUDAGuard guard(x.device());
        out = heads_out(args[5], x, "out");
        TORCH_CHECK(!overlap(out, x) || (same_place(out, x) && layout != GPUK_ROPE_SPLIT), "gpuk: rope: out overlaps x");
        check(gpuk_rope(x.const_data_ptr(), stride_of(x, 0), stride_of(x, 1), out.data_ptr(), stride_of(out, 0), stride_of(out, 1), pos.data_ptr<int64_t>(), turns.data_ptr<int64_t>(),
                        static_cast<float>(amplitude), int_size(x.size(0)), int_size(x.size(1)), int_size(x.size(2)), int_size(2 * turns.numel()), int_size(layout), dtype_of(x, "x"),
                        stream_of(x)), "rope");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// rope_paged(q, k, v, positions, slots, turns, amplitude, layout, k_pages, v_pages, out or None) -> rotated queries
PyObject *rope_paged(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect_args(n, 11, "rope_paged");
    expect_unwatched("rope_paged");
    const Tensor &q = heads_arg(args[0], "q", -1);
    const int dev = q.get_device();
    const Tensor &k = heads_arg(args[1], "k", dev), &v = heads_arg(args[2], "v", dev);
    const int64_t tokens = q.size(0);
    const Tensor &pos = ints_arg(args[3], "positions", dev, at::kLong, tokens), &slots = ints_arg(args[4], "slots", dev, at::kLong, tokens), &turns = paged_arg(args[5], "frequencies", dev);
    ints_arg(args[5], "frequencies", dev, at::kLong, turns.numel());
    const double amplitude = float_arg(args[6]);
    const int64_t layout = int_arg(args[7]);
    const Pages pages(args[8], args[9], dev, false, true);
    TORCH_CHECK(k.size(0) == tokens && v.sizes() == k.sizes() && k.size(1) == pages.c.kv_heads && k.size(2) == pages.c.head_dim && q.size(2) == pages.c.head_dim,
                "gpuk: rope_paged shapes do not match");
    TORCH_CHECK(q.scalar_type() == pages.k.scalar_type() && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), "gpuk: rope_paged takes one type");
    Tensor out;
    {
        NoGil unlocked;
        c10::cuda::CUDAGuard guard(q.device());
        out = heads_out(args[10], q, "out");
        TORCH_CHECK((!overlap(out, q) || (same_place(out, q) && layout != GPUK_ROPE_SPLIT)), "gpuk: rope_paged: out overlaps q");
        for (const Tensor *t : std::initializer_list<const Tensor *>{&out, &q, &k, &v}) TORCH_CHECK(!overlap(*t, pages.k) && !overlap(*t, pages.v), "gpuk: rope_paged: a tensor overlaps the pages");
        TORCH_CHECK(!overlap(out, k) && !overlap(out, v), "gpuk: rope_paged: out overlaps k or v");
        check(gpuk_rope_paged(q.const_data_ptr(), stride_of(q, 0), stride_of(q, 1), k.const_data_ptr(), stride_of(k, 0), stride_of(k, 1), v.const_data_ptr(), stride_of(v, 0),
                              stride_of(v, 1), out.data_ptr(), stride_of(out, 0), stride_of(out, 1), pos.data_ptr<int64_t>(), slots.data_ptr<int64_t>(), turns.data_ptr<int64_t>(),
                              static_cast<float>(amplitude), &pages.c, int_size(tokens), int_size(q.size(1)), int_size(2 * turns.numel()), int_size(layout), stream_of(q)),
              "rope_paged");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// paged_attention(q [tokens, heads, head_dim], k_pages, v_pages, tables, lens, starts, masks or None, max_len (negative: what the table holds), max_new (0: not known),
// scale (0: 1 / sqrt(head_dim)), out or None)
PyObject *paged_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect_args(n, 11, "paged_attention");
    expect_unwatched("paged_attention");
    const Tensor &q = heads_arg(args[0], "q", -1);
    const int dev = q.get_device();
    const Pages pages(args[1], args[2], dev, false, false);
    const Tensor &lens = paged_arg(args[4], "lens", dev);
    TORCH_CHECK(lens.dim() == 1, "gpuk: lens must be one-dimensional");
    const int64_t batch = lens.size(0), tokens = q.size(0);
    ints_arg(args[4], "lens", dev, at::kInt, batch);
    const Tensor &tables = rows_arg(args[3], "tables", dev, batch), &starts = ints_arg(args[5], "starts", dev, at::kInt, batch + 1);
    const Tensor *masks = nullptr;
    if (args[6] != Py_None) {
        masks = &rows_arg(args[6], "masks", dev, tokens);
        TORCH_CHECK(masks->is_contiguous() && masks->size(1) >= 1, "gpuk: masks must be contiguous, with a word or more");
    }
    int64_t max_len = int_arg(args[7]);
    const int max_new = int_size(int_arg(args[8]));
    double scale = float_arg(args[9]);
    TORCH_CHECK(q.size(2) == pages.c.head_dim && q.scalar_type() == pages.k.scalar_type(), "gpuk: paged_attention: q and the pages have different heads or types");
    if (scale == 0.0) scale = 1.0 / std::sqrt(static_cast<double>(std::max<int64_t>(1, q.size(2))));
    const int64_t holds = tables.size(1) * pages.c.page_size;
    if (max_len < 0 || max_len > holds) max_len = holds;
    Tensor out;
    {
        NoGil unlocked;
        c10::cuda::CUDAGuard guard(q.device());
        out = heads_out(args[10], q, "out");
        TORCH_CHECK(!overlap(out, q) && !overlap(out, pages.k) && !overlap(out, pages.v), "gpuk: paged_attention: out overlaps what is read");
        int64_t bytes = 0;
        check(gpuk_paged_attention_workspace(&pages.c, int_size(batch), int_size(tokens), int_size(q.size(1)), max_len, &bytes), "paged_attention");
        // of the call's own: freed to the allocator on its stream, so two captured graphs never share one
        Tensor workspace;
        if (bytes) workspace = empty_like_on(q, {bytes}, at::kByte);
        check(gpuk_paged_attention(q.const_data_ptr(), stride_of(q, 0), stride_of(q, 1), &pages.c, tables.data_ptr<int>(), batch > 1 ? tables.stride(0) : tables.size(1),
                                   int_size(tables.size(1)), lens.data_ptr<int>(), starts.data_ptr<int>(), masks ? masks->data_ptr<int>() : nullptr, masks ? int_size(masks->size(1)) : 0,
                                   out.data_ptr(), stride_of(out, 0), stride_of(out, 1), int_size(batch), int_size(tokens), int_size(q.size(1)), max_len, max_new, static_cast<float>(scale),
                                   bytes ? workspace.data_ptr() : nullptr, bytes, stream_of(q)), "paged_attention");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// paged_keep(k_pages, v_pages, tables, lens, paths [batch, depth], held or None, out or None) -> lens
PyObject *paged_keep(PyObject *, PyObject *const *args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    expect_args(n, 7, "paged_keep");
    expect_unwatched("paged_keep");
    const Pages pages(args[0], args[1], -1, true, true);
    const int dev = pages.k.get_device();
    const Tensor &lens = paged_arg(args[3], "lens", dev);
    TORCH_CHECK(lens.dim() == 1, "gpuk: lens must be one-dimensional");
    const int64_t batch = lens.size(0);
    ints_arg(args[3], "lens", dev, at::kInt, batch);
    const Tensor &tables = rows_arg(args[2], "tables", dev, batch), &paths = rows_arg(args[4], "paths", dev, batch);
    const Tensor *held = args[5] == Py_None ? nullptr : &ints_arg(args[5], "held", dev, at::kInt, batch);
    Tensor out;
    if (args[6] != Py_None) {
        out = ints_arg(args[6], "out", dev, at::kInt, batch);
        for (const Tensor *t : {&lens, &tables, &paths, held}) TORCH_CHECK(!t || !overlap(out, *t), "gpuk: paged_keep: out overlaps what is read");
    }
    {
        NoGil unlocked;
        c10::cuda::CUDAGuard guard(pages.k.device());
        if (!out.defined()) out = empty_like_on(lens, {batch}, at::kInt);
        check(gpuk_paged_keep_held(&pages.c, int_size(pages.layers), pages.layer_stride, tables.data_ptr<int>(), batch > 1 ? tables.stride(0) : tables.size(1), int_size(tables.size(1)),
                                   lens.data_ptr<int>(), paths.data_ptr<int>(), batch > 1 ? paths.stride(0) : paths.size(1), int_size(paths.size(1)),
                                   held ? held->data_ptr<int>() : nullptr, out.data_ptr<int>(), int_size(batch), stream_of(lens)), "paged_keep");
    }
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

}  // namespace gpuk_native
