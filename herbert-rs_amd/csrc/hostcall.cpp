// The host's side of a launch, natively: the check that every operand of every kernel passes, and the call of a module's C
// entry point. A step that is not a graph's replay makes one call a kernel with 15 to 30 arguments and checks five operands for
// each; in Python (attribute after attribute, a generator over a shape) and through ctypes (an object an argument) that took 9 of the 16
// microseconds that a launch costs the host, longer than most kernels of a short prompt run. A check takes 0.09 us here instead of 0.66,
// a call of 24 arguments that its entry point refuses 0.9 instead of 1.8. And the plan of a step whose sequences share pages, which
// changes wherever one of them begins a page.
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdint.h>

#include <algorithm>
#include <exception>
#include <vector>

#if !defined(__x86_64__) || !defined(__linux__)
#error "entry points are called as the x86-64 System V calling convention passes their arguments"
#endif

namespace {

// What is called. Every entry point takes pointers, integers and up to FLOATS floats and returns int. The calling convention passes
// integers and pointers in one sequence (six registers, then the stack, eight bytes each) and floats in another
// (eight registers), so any such function can be called as one that takes all floats first and more integers than it has:
// it finds its own where it looks, and the caller takes the rest off the stack again.
constexpr int FLOATS = 8, WORDS = 40;
#define W8 uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t
typedef int (*Function)(float, float, float, float, float, float, float, float, W8, W8, W8, W8, W8);

struct Entry {
    Function function;
    int count;
    bool is_float[WORDS + FLOATS];
};
const char ENTRY[] = "herbert_rs_amd.entry";

void free_entry(PyObject* capsule) { delete (Entry*)PyCapsule_GetPointer(capsule, ENTRY); }

// entry(address, kinds): kinds has a letter an argument, 'f' for a float and 'i' for anything else.
PyObject* make_entry(PyObject*, PyObject* args) {
    unsigned long long address;
    const char* kinds;
    if (!PyArg_ParseTuple(args, "Ks", &address, &kinds)) return nullptr;
    int words = 0, floats = 0;
    Entry e;
    e.function = (Function)address;
    e.count = 0;
    for (; kinds[e.count]; ++e.count) {
        const bool f = kinds[e.count] == 'f';
        if ((f ? ++floats : ++words) > (f ? FLOATS : WORDS)) {
            PyErr_SetString(PyExc_ValueError, "an entry point with more arguments than are passed on");
            return nullptr;
        }
        e.is_float[e.count] = f;
    }
    return PyCapsule_New(new Entry(e), ENTRY, free_entry);
}

// invoke(entry, arguments...): what the function returns. None is a null pointer, a tensor its memory; the interpreter is free meanwhile.
PyObject* invoke(PyObject*, PyObject* const* args, Py_ssize_t n) {
    Entry* e = n > 0 ? (Entry*)PyCapsule_GetPointer(args[0], ENTRY) : nullptr;
    if (!e) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "an entry point is needed");
        return nullptr;
    }
    if (n - 1 != e->count) return PyErr_Format(PyExc_TypeError, "the entry point takes %d arguments, not %zd", e->count, n - 1);
    float f[FLOATS] = {};
    uint64_t w[WORDS] = {};
    int nf = 0, nw = 0;
    for (int i = 0; i < e->count; ++i) {
        PyObject* a = args[1 + i];
        if (e->is_float[i]) {
            f[nf++] = (float)PyFloat_AsDouble(a);
        } else if (a == Py_None) {
            w[nw++] = 0;
        } else if (!PyLong_Check(a) && THPVariable_Check(a)) {
            try {
                w[nw++] = (uint64_t)THPVariable_Unpack(a).data_ptr();
            } catch (const std::exception& ex) {
                return PyErr_Format(PyExc_TypeError, "argument %d has no memory: %s", i, ex.what());
            }
        } else {
            w[nw++] = PyLong_AsUnsignedLongLongMask(a);
        }
    }
    if (PyErr_Occurred()) return nullptr;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = e->function(f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7], w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9],
                     w[10], w[11], w[12], w[13], w[14], w[15], w[16], w[17], w[18], w[19], w[20], w[21], w[22], w[23], w[24],
                     w[25], w[26], w[27], w[28], w[29], w[30], w[31], w[32], w[33], w[34], w[35], w[36], w[37], w[38], w[39]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

bool has_form(const at::Tensor& t, PyObject* dtype, PyObject* shape) {
    if (!t.is_cuda() || !t.is_contiguous()) return false;
    if (dtype != Py_None && (!THPDtype_Check(dtype) || ((THPDtype*)dtype)->scalar_type != t.scalar_type())) return false;
    if (shape == Py_None) return true;
    if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != t.dim()) return false;
    for (int64_t i = 0; i < t.dim(); ++i) {
        PyObject* want = PyTuple_GET_ITEM(shape, i);
        if (want == Py_None) continue;
        const long long size = PyLong_AsLongLong(want);
        if ((size == -1 && PyErr_Occurred()) || size != t.size(i)) return false;
    }
    return true;
}

// fits(tensor, dtype or None, shape or None): True for a contiguous tensor on the GPU of that type and shape (None within the
// shape: any size). Anything else is False, and the caller says what is wrong; also a tensor that throws where it is asked (a sparse one
// or a subclass has no strides to look at): an exception of C++ must not leave a function that the interpreter called.
PyObject* fits(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 3) {
        PyErr_SetString(PyExc_TypeError, "a tensor, a type and a shape are needed");
        return nullptr;
    }
    bool is = false;
    try {
        is = THPVariable_Check(args[0]) && has_form(THPVariable_Unpack(args[0]), args[1], args[2]);
    } catch (const std::exception&) {
    }
    PyErr_Clear();
    return PyBool_FromLong(is);
}

// all_fit(tensor, dtype, shape, tensor, dtype, shape, ...): the GPU that all of them lie on if each fits, else -1, and the caller says
// what is wrong.
PyObject* all_fit(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n % 3 != 0) {
        PyErr_SetString(PyExc_TypeError, "tensors, each with a type and a shape, are needed");
        return nullptr;
    }
    long at = -1;
    bool is = true;
    try {
        for (Py_ssize_t i = 0; is && i < n; i += 3) {
            is = THPVariable_Check(args[i]) && has_form(THPVariable_Unpack(args[i]), args[i + 1], args[i + 2]);
            if (!is) break;
            const long device = THPVariable_Unpack(args[i]).get_device();
            is = at < 0 || at == device;
            at = device;
        }
    } catch (const std::exception&) {
        is = false;
    }
    PyErr_Clear();
    return PyLong_FromLong(is ? at : -1);
}

// A contiguous array of 64-bit integers that the caller holds.
class Numbers {
  public:
    Numbers() = default;
    Numbers(const Numbers&) = delete;
    ~Numbers() {
        if (view_.obj) PyBuffer_Release(&view_);
    }
    bool take(PyObject* from, const char* what) {
        if (PyObject_GetBuffer(from, &view_, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT) != 0) return false;
        if (view_.itemsize != 8 || !view_.format || (view_.format[0] != 'l' && view_.format[0] != 'q') || view_.format[1]) {
            PyErr_Format(PyExc_TypeError, "%s must be 64-bit integers", what);
            return false;
        }
        return true;
    }
    int64_t size() const { return view_.len / 8; }
    int64_t operator[](int64_t i) const { return ((const int64_t*)view_.buf)[i]; }

  private:
    Py_buffer view_{};
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Tile {
    int64_t row0, rows, seq, page, end, whole;
};
constexpr int ITEM_INTS = 8;
struct PlanItem {
    int32_t row0, rows, slot, page0, page1, list0, masked, unused;
};

// The cut of kernels/shared.py's plan, which says what it is. Returns false where the arrays do not describe a step (nothing outside them is
// read, and what is made stays within a step's size).
bool cut_plan(const Numbers& starts, const Numbers& context, const Numbers& slots, const Numbers& order, const Numbers& nodes, int64_t group,
              int64_t nkv, int64_t columns, int64_t masked_columns, int64_t workgroups, int64_t grid, int64_t room, std::vector<int32_t>& out,
              int64_t& n_items, int64_t& n_parts, int64_t& most) {
    const int64_t B = order.size(), T = B > 0 && starts.size() == B + 1 ? starts[B] - starts[0] : 0;
    if (T <= 0 || T > INT32_MAX || starts[0] != 0 || context.size() != B || slots.size() != B || nodes.size() % 4 || group <= 0 || nkv <= 0 ||
        columns <= 0 || masked_columns <= 0 || workgroups <= 0 || grid <= 0 || room < 0 || room > INT32_MAX)
        return false;
    std::vector<int64_t> row_of(B + 1, 0);                // a sequence's first row in the order
    std::vector<int32_t> rows_in_order;
    std::vector<bool> met(B, false);
    rows_in_order.reserve(T);
    for (int64_t i = 0; i < B; ++i) {
        const int64_t seq = order[i];
        if (seq < 0 || seq >= B || met[seq] || starts[seq + 1] <= starts[seq] || context[seq] < starts[seq + 1] - starts[seq] ||
            context[seq] > INT32_MAX)
            return false;
        met[seq] = true;
        row_of[i + 1] = row_of[i] + starts[seq + 1] - starts[seq];
        for (int64_t r = starts[seq]; r < starts[seq + 1]; ++r) rows_in_order.push_back((int32_t)r);
    }
    const int64_t tall = std::max<int64_t>(1, columns / group);
    const int64_t low = columns == 128 ? std::max<int64_t>(1, masked_columns / group) : tall;
    std::vector<Tile> tiles;
    auto even = [](int64_t first, int64_t end, int64_t most_rows, auto f) {
        const int64_t count = ceil_div(end - first, most_rows);
        for (int64_t i = 0; i < count; ++i) {
            const int64_t from = first + (end - first) * i / count, to = first + (end - first) * (i + 1) / count;
            f(from, to - from);
        }
    };
    auto is_alone = [&](int64_t k) { return nodes[4 * k + 3] < 0 && row_of[nodes[4 * k] + 1] - row_of[nodes[4 * k]] == 1; };
    const int64_t n_nodes = nodes.size() / 4;
    std::vector<int64_t> covered(B, 0);                   // pages of the sequences in the order that nodes so far hold; -1: all
    for (int64_t k = 0; k < n_nodes; ++k) {
        const int64_t first = nodes[4 * k], count = nodes[4 * k + 1], page = nodes[4 * k + 2], end = nodes[4 * k + 3];
        if (first < 0 || count <= 0 || count > B || first + count > B || page < 0 || page > INT32_MAX || end > INT32_MAX || (end < 0 && count != 1) ||
            (end >= 0 && end <= page))
            return false;
        for (int64_t i = first; i < first + count; ++i) {  // (shared pages lie before what the step brings)
            if (covered[i] != page || (end >= 0 && 64 * end > context[order[i]] - (row_of[i + 1] - row_of[i]) + 1)) return false;
            covered[i] = end;
        }
        if (is_alone(k)) continue;                        // (a sequence's own pages, one row: behind the others)
        const int64_t a = row_of[first], b = row_of[first + count], seq = order[first], held = context[seq];
        even(a, b, tall, [&](int64_t r, int64_t n) {
            if (end >= 0) {
                tiles.push_back({r, n, seq, page, end, end});
                return;
            }
            // A sequence's own rows: all of them see what lies before the first row's page; a tile ends at the page of its last row.
            const int64_t whole = (held - (b - r)) / 64;
            int64_t from = page;
            if (n * group > 64 && whole > page) {
                tiles.push_back({r, n, seq, page, whole, whole});
                from = whole;
            }
            even(r, r + n, low, [&](int64_t u, int64_t m) {
                tiles.push_back({u, m, seq, from, (held - (b - (u + m)) - 1) / 64 + 1, (held - (b - u)) / 64});
            });
        });
    }
    for (int64_t k = 0; k < n_nodes; ++k)
        if (is_alone(k)) {
            const int64_t first = nodes[4 * k], seq = order[first], seen = (context[seq] - 1) / 64;
            tiles.push_back({row_of[first], 1, seq, nodes[4 * k + 2], seen + 1, seen});
        }
    for (int64_t i = 0; i < B; ++i)
        if (covered[i] >= 0) return false;
    int64_t all_pages = 0;
    for (const Tile& t : tiles) {
        if (t.end <= t.page) return false;
        all_pages += t.end - t.page;
    }
    const int64_t share = std::max<int64_t>(1, ceil_div(all_pages * nkv, workgroups));
    std::vector<PlanItem> items;
    std::vector<int32_t> begins(T + 1, 0);                // of a row's partial results
    most = 0;
    n_parts = 0;
    for (const Tile& t : tiles) {
        const int64_t cols = t.rows * group, turns = columns != 128 ? 1 : cols <= 32 ? 4 : cols <= 64 ? 2 : 1;
        int64_t per = ceil_div(share, turns) * turns;
        const int64_t ranges = ceil_div(t.end - t.page, per);
        per = ceil_div(ceil_div(t.end - t.page, ranges), turns) * turns;
        for (int64_t page = t.page; page < t.end; page += per) {
            const int64_t to = std::min(page + per, t.end);
            items.push_back({(int32_t)t.row0, (int32_t)t.rows, (int32_t)slots[t.seq], (int32_t)page, (int32_t)to, (int32_t)n_parts, to > t.whole, 0});
            n_parts += t.rows;
            if (n_parts > INT32_MAX) return false;
            for (int64_t r = 0; r < t.rows; ++r) ++begins[t.row0 + r + 1];
        }
        most = std::max(most, t.rows);
    }
    for (int64_t r = 0; r < T; ++r) begins[r + 1] += begins[r];
    n_items = ceil_div((int64_t)items.size(), grid) * grid;
    room = std::max(room, n_items);
    out.assign(ITEM_INTS * room + T + T + 1 + n_parts, 0);
    int32_t* const order_at = out.data() + ITEM_INTS * room;
    std::copy(rows_in_order.begin(), rows_in_order.end(), order_at);
    std::copy(begins.begin(), begins.end(), order_at + T);
    // a row's partial results lie side by side, in the order of its items
    int32_t* const parts = order_at + 2 * T + 1;
    for (const PlanItem& it : items)
        for (int32_t r = 0; r < it.rows; ++r) parts[it.list0 + r] = begins[it.row0 + r]++;
    // the longest items first, those over the same pages side by side
    std::stable_sort(items.begin(), items.end(), [](const PlanItem& x, const PlanItem& y) {
        const int32_t n = x.page1 - x.page0, m = y.page1 - y.page0;
        return n != m ? n > m : x.page0 != y.page0 ? x.page0 < y.page0 : x.row0 < y.row0;
    });
    static_assert(sizeof(PlanItem) == ITEM_INTS * sizeof(int32_t), "an item is ITEM_INTS numbers");
    std::copy((const int32_t*)items.data(), (const int32_t*)(items.data() + items.size()), out.data());
    return true;
}

// plan(starts, context, slots, order, nodes, group, kv heads, columns, masked columns, workgroups, grid, room): (the items, in the room of so many at
// least, the order of the rows, where their partial results begin and the places of the items' rows among them, one after another as
// 32-bit numbers; how many items, how many places, the most rows of an item), or None where the arrays do not describe a step.
PyObject* plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 12) {
        PyErr_SetString(PyExc_TypeError, "five arrays and seven numbers are needed");
        return nullptr;
    }
    Numbers arrays[5];
    const char* const names[5] = {"starts", "context", "slots", "order", "nodes"};
    for (int i = 0; i < 5; ++i)
        if (!arrays[i].take(args[i], names[i])) return nullptr;
    int64_t numbers[7];
    for (int i = 0; i < 7; ++i) numbers[i] = PyLong_AsLongLong(args[5 + i]);
    if (PyErr_Occurred()) return nullptr;
    std::vector<int32_t> out;
    int64_t n_items = 0, n_parts = 0, most = 0;
    try {
        if (!cut_plan(arrays[0], arrays[1], arrays[2], arrays[3], arrays[4], numbers[0], numbers[1], numbers[2], numbers[3], numbers[4], numbers[5],
                      numbers[6], out, n_items, n_parts, most))
            Py_RETURN_NONE;
    } catch (const std::exception& e) {
        return PyErr_Format(PyExc_MemoryError, "a plan of shared pages: %s", e.what());
    }
    PyObject* bytes = PyByteArray_FromStringAndSize((const char*)out.data(), (Py_ssize_t)(4 * out.size()));
    return bytes ? Py_BuildValue("NLLL", bytes, (long long)n_items, (long long)n_parts, (long long)most) : nullptr;
}

PyMethodDef methods[] = {{"entry", make_entry, METH_VARARGS, nullptr},
                         {"invoke", (PyCFunction)(void*)invoke, METH_FASTCALL, nullptr},
                         {"fits", (PyCFunction)(void*)fits, METH_FASTCALL, nullptr},
                         {"all_fit", (PyCFunction)(void*)all_fit, METH_FASTCALL, nullptr},
                         {"plan", (PyCFunction)(void*)plan, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "hostcall", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_hostcall() { return PyModule_Create(&module); }
