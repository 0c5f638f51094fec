// graph_host.cpp — a minimal ggml-like host for the plugin (test infrastructure only): the base functions
// that the plugin resolves from the process that loaded it, and enough to build a graph by hand and run it
// on the first device. Tests load it with ctypes (RTLD_GLOBAL) before the plugin:
//   gh_open(plugin)                                   1 when a backend came up
//   gh_tensor(op, type, ne, nb, data, src, n_src, params, n_params) -> index of the new tensor
//   gh_view(t, of, offset)                            t becomes a view without data yet
//   gh_supports(t)                                    supports_op of the device
//   gh_graph(nodes, n)  gh_compute() -> ggml_status   one graph at a time; compute waits for the result
#include "../ggml-gfx906_amd/csrc/ggml_abi.h"

#include <dlfcn.h>

#include <cstring>
#include <deque>
#include <vector>

#define API extern "C" __attribute__((visibility("default")))

API ggml_backend_buffer_t ggml_backend_buffer_init(ggml_backend_buffer_type_t buft, struct ggml_backend_buffer_i iface, void *ctx, size_t size) {
    auto *b = new ggml_backend_buffer();
    b->iface = iface;
    b->buft = buft;
    b->context = ctx;
    b->size = size;
    return b;
}
API int ggml_graph_n_nodes(struct ggml_cgraph *g) { return g->n_nodes; }
API struct ggml_tensor *ggml_graph_node(struct ggml_cgraph *g, int i) { return g->nodes[i < 0 ? g->n_nodes + i : i]; }
API size_t ggml_nbytes(const struct ggml_tensor *t) {   // (value types only: the blocks of quantized rows are not looked at)
    size_t n = t->type == GGMLABI_TYPE_F32 || t->type == GGMLABI_TYPE_I32 ? 4 : 2;
    for (int i = 0; i < 4; ++i) {
        if (t->ne[i] <= 0) return 0;
        n += (size_t)(t->ne[i] - 1) * t->nb[i];
    }
    return n;
}

namespace {
std::deque<ggml_tensor> tensors;
std::vector<ggml_tensor *> nodes, keys;
std::vector<int32_t> uses;
std::vector<uint32_t> used;
ggml_cgraph graph;
ggml_backend_t backend;
ggml_backend_dev_t device;

size_t slot_of(ggml_tensor *t) {
    size_t i = ((size_t)(uintptr_t)t >> 4) % keys.size();
    while ((used[i >> 5] & (1u << (i & 31))) && keys[i] != t) i = (i + 1) % keys.size();
    return i;
}
}  // namespace

API int gh_open(const char *plugin) {
    if (backend) return 1;
    void *h = dlopen(plugin, RTLD_NOW | RTLD_GLOBAL);
    if (!h) return 0;
    auto init = reinterpret_cast<ggml_backend_reg_t (*)()>(dlsym(h, "ggml_backend_init"));
    ggml_backend_reg_t reg = init ? init() : nullptr;
    if (!reg || reg->iface.get_device_count(reg) == 0) return 0;
    device = reg->iface.get_device(reg, 0);
    backend = device->iface.init_backend(device, nullptr);
    return backend != nullptr;
}

API int gh_tensor(int op, int type, const int64_t *ne, const size_t *nb, void *data, const int *src, int n_src, const int32_t *params, int n_params) {
    ggml_tensor t;
    std::memset(&t, 0, sizeof t);
    t.op = op;
    t.type = type;
    t.data = data;
    for (int i = 0; i < 4; ++i) {
        t.ne[i] = ne[i];
        t.nb[i] = nb[i];
    }
    for (int i = 0; i < n_src; ++i) t.src[i] = src[i] < 0 ? nullptr : &tensors[src[i]];
    std::memcpy(t.op_params, params, n_params * sizeof(int32_t));
    tensors.push_back(t);
    return (int)tensors.size() - 1;
}

API void gh_view(int t, int of, size_t offset) {
    tensors[t].data = nullptr;
    tensors[t].view_src = &tensors[of];
    tensors[t].view_offs = offset;
}

API int gh_supports(int t) { return device->iface.supports_op(device, &tensors[t]); }

API void gh_graph(const int *list, int n) {
    nodes.clear();
    keys.assign(4 * tensors.size() + 7, nullptr);
    used.assign(keys.size() / 32 + 1, 0);
    uses.assign(keys.size(), 0);
    auto add = [](ggml_tensor *t) {
        const size_t i = slot_of(t);
        keys[i] = t;
        used[i >> 5] |= 1u << (i & 31);
        return i;
    };
    for (int i = 0; i < n; ++i) {
        nodes.push_back(&tensors[list[i]]);
        add(nodes.back());
        for (ggml_tensor *s : nodes.back()->src)
            if (s) ++uses[add(s)];
    }
    std::memset(&graph, 0, sizeof graph);
    graph.size = graph.n_nodes = n;
    graph.nodes = nodes.data();
    graph.use_counts = uses.data();
    graph.visited_hash_set = {keys.size(), used.data(), keys.data()};
}

API int gh_compute() {
    const int st = backend->iface.graph_compute(backend, &graph);
    backend->iface.synchronize(backend);
    return st;
}
