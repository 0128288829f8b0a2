// extern "C" surface of the operators that run on a stream of the caller's choice (part 4 of include/cpmcu_b200.h): 8-bit linear
// layers and rotations.  They launch and return: no allocation, no synchronisation, no host copy.
#include <algorithm>
#include <climits>
#include <initializer_list>

#include "../../include/cpmcu_b200.h"
#include "op_errors.cuh"
#include "rotary.cuh"
#include "w8a8.cuh"

namespace {

template <typename F>
auto guarded(F&& f) -> decltype(f()) {
    try {
        cpm_set_error("");
        return f();
    } catch (const std::exception& e) {
        cpm_set_error(e.what());
        return -1;
    } catch (...) {
        cpm_set_error("unknown error");
        return -1;
    }
}

// The message is put together only where it is needed.
void require(bool ok, const char* what, const char* msg) {
    if (!ok) throw std::invalid_argument(std::string("cpmcu_b200: ") + what + ": " + msg);
}

uintptr_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Rows of `cols` elements of `size` bytes, `ld` elements apart.
struct Rows {
    const void* p;
    long long rows, cols, ld;
    int size;
    uintptr_t end() const { return addr(p) + static_cast<uintptr_t>(((rows - 1) * ld + cols) * size); }
};
// Whether two sets of rows share an element.  Columns of one wider matrix do not, although their rows interleave.
bool overlap(const Rows& a, const Rows& b) {
    if (a.p == nullptr || b.p == nullptr || a.rows < 1 || b.rows < 1 || a.end() <= addr(b.p) || b.end() <= addr(a.p)) return false;
    const long long pitch = a.ld * a.size;
    if (a.rows > 1 && b.rows > 1 && pitch == b.ld * b.size) {
        const bool a_first = addr(a.p) <= addr(b.p);
        const Rows &lo = a_first ? a : b, &hi = a_first ? b : a;
        const long long off = static_cast<long long>((addr(hi.p) - addr(lo.p)) % static_cast<uintptr_t>(pitch));
        if (off >= lo.cols * lo.size && off + hi.cols * hi.size <= pitch) return false;
    }
    return true;
}

Rows whole(const void* p, size_t bytes) { return {p, 1, static_cast<long long>(bytes), static_cast<long long>(bytes), 1}; }

// The library serves the GPU that was current at its first call (one process per GPU).
void require_device(const char* what) {
    int device = -1;
    CUDA_CHECK(cudaGetDevice(&device));
    if (device != runtime().device) {
        throw std::invalid_argument(std::string("cpmcu_b200: ") + what + ": the current device is " + std::to_string(device) +
                                    ", the library runs on device " + std::to_string(runtime().device));
    }
}

cudaStream_t stream_of(void* s) { return static_cast<cudaStream_t>(s); }

void require_sizes(const char* what, int rows, int N, int K) {
    require(rows >= 0 && N >= 1 && K >= 1, what, "sizes must be positive");
    require(K <= w8::MAX_COLS, what, "sums of more than 131072 products do not fit 32 bits");
    const long long tiles = (static_cast<long long>(N) + 63) / 64;
    require(tiles * (w8::pad_cols(K) / w8::BLOCK_COLS) <= (1ll << 23) && ((static_cast<long long>(rows) + 15) / 16) * tiles <= (1ll << 30), what, "too many tiles");
}
// Products count rows in whole token tiles, of up to 256, and in 32 bits.
void require_rows(const char* what, int rows) { require(rows <= INT_MAX - 256, what, "too many rows"); }

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

// A call's workspace: what is where.  Nothing in it is kept from one call for the next.
struct Layout {
    size_t q = 0, xs = 0, tickets = 0, partials = 0, act = 0, total = 0;
    int n_tickets = 0;
    long long act_ld = 0;
};
Layout layout_of(int rows, int N, int K, int inter) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += align256(bytes); return here; };
    if (inter > 0) {
        l.act_ld = (inter + 7) / 8 * 8;
        l.act = take(static_cast<size_t>(rows) * l.act_ld * sizeof(float));
    }
    if (rows > 1) {
        l.q = take(static_cast<size_t>(rows) * std::max(w8::pad_cols(K), inter > 0 ? w8::pad_cols(inter) : 0));
        l.xs = take(align256(rows) * sizeof(float));
        // the down projection's, or the only product's
        const w8::Scratch scratch = w8::product_scratch(rows, N, inter > 0 ? inter : K);
        l.n_tickets = scratch.tickets;
        l.tickets = take(l.n_tickets * sizeof(int));
        l.partials = take(scratch.partial_bytes);
    }
    l.total = at;
    return l;
}

w8::RowSource source_of(const char* what, const void* x, long long ldx, const void* norm, float eps, const void* delta, float delta_scale, void* total,
                        int rows, int K, const void* y, long long ldy, int out) {
    require(x != nullptr && y != nullptr, what, "x and y must not be null");
    require(ldx >= K && ldy >= out, what, "rows overlap: a leading dimension is smaller than the row");
    require(ldy < (1ll << 31), what, "the leading dimension of y does not fit 32 bits");
    require(norm != nullptr || delta == nullptr, what, "a delta needs the norm's weights");
    require((delta == nullptr) == (total == nullptr), what, "delta and total come together");
    w8::RowSource s;
    s.x = static_cast<const bf16*>(x);
    s.ldx = ldx;
    const Rows xr{x, rows, K, ldx, 2}, yr{y, rows, out, ldy, 2};
    require(!overlap(xr, yr), what, "y must not overlap x");
    if (norm != nullptr) {
        s.norm = static_cast<const bf16*>(norm);
        s.eps = eps;
        s.delta = static_cast<const bf16*>(delta);
        s.total = static_cast<bf16*>(total);
        s.delta_scale = delta_scale;
        const Rows dr{delta, rows, K, K, 2}, tr{total, rows, K, K, 2}, wr{norm, 1, K, K, 2};
        require(!overlap(tr, xr) && !overlap(tr, dr) && !overlap(tr, yr) && !overlap(tr, wr), what, "total must not overlap x, delta, y or the weights");
        require(!overlap(yr, dr) && !overlap(yr, wr), what, "y must not overlap delta or the weights");
    }
    return s;
}

// The workspace, and that it shares nothing with what the call reads and writes.
void require_workspace(const char* what, void* ws, long long bytes, const Layout& l, std::initializer_list<Rows> others) {
    if (l.total == 0) return;
    if (ws == nullptr || bytes < 0 || static_cast<size_t>(bytes) < l.total) {
        throw std::invalid_argument(std::string("cpmcu_b200: ") + what + ": the workspace needs " + std::to_string(l.total) + " bytes");
    }
    require((addr(ws) & 255) == 0, what, "the workspace must be 256-byte aligned");
    const Rows wr = whole(ws, l.total);
    for (const Rows& o : others) require(!overlap(wr, o), what, "the workspace must not overlap what the call reads or writes");
}
// What the call writes shares nothing with the weights and the bias.
void require_apart(const char* what, std::initializer_list<Rows> written, std::initializer_list<Rows> constant) {
    for (const Rows& w : written) {
        for (const Rows& c : constant) require(!overlap(w, c), what, "y and total must not overlap the weights or the bias");
    }
}

void require_packed(const char* what, const void* packed) {
    require(packed != nullptr && (addr(packed) & 255) == 0, what, "packed weights must be 256-byte aligned");
}

}  // namespace

extern "C" {

int cpmcu_stream_check(void* stream) {
    return guarded([&] {
        require_device("stream_check");
        const OpErrors e = new_op_errors(stream_of(stream));
        if ((e.own | e.shared) != 0) {
            throw std::runtime_error("cpmcu_b200: kernel error flags " + std::to_string(e.own | e.shared) +
                                     (e.shared != 0 ? ", of launches of captured graphs, on this stream or another one, " + std::to_string(e.shared) : ""));
        }
        return 0;
    });
}

long cpmcu_w8a8_packed_bytes(int N, int K, int gated) {
    return guarded([&]() -> long {
        require_sizes("w8a8_packed_bytes", 1, N, K);
        return static_cast<long>(w8::packed_bytes(N, K, gated != 0));
    });
}

int cpmcu_w8a8_pack(const void* q, const float* scale, int N, int K, int part, void* packed, void* stream) {
    return guarded([&] {
        require_sizes("w8a8_pack", 1, N, K);
        CPM_REQUIRE(q != nullptr && scale != nullptr, "w8a8_pack: q and scale must not be null");
        CPM_REQUIRE(part >= 0 && part <= 2, "w8a8_pack: part is 0, 1 (gate) or 2 (up)");
        require_packed("w8a8_pack", packed);
        const Rows pr = whole(packed, w8::packed_bytes(N, K, part != 0));
        CPM_REQUIRE(!overlap(pr, whole(q, static_cast<size_t>(N) * K)) && !overlap(pr, whole(scale, static_cast<size_t>(N) * 4)), "w8a8_pack: packed must not overlap q or scale");
        require_device("w8a8_pack");
        w8::launch_pack(static_cast<const int8_t*>(q), scale, N, K, static_cast<w8::Role>(part), packed, stream_of(stream));
        return 0;
    });
}

int cpmcu_w8a8_quantize(const void* x, long long ldx, int rows, int K, void* q, float* scale, void* stream) {
    return guarded([&] {
        require_sizes("w8a8_quantize", rows, 1, K);
        if (rows == 0) return 0;
        CPM_REQUIRE(x != nullptr && q != nullptr && scale != nullptr, "w8a8_quantize: x, q and scale must not be null");
        CPM_REQUIRE(ldx >= K, "w8a8_quantize: rows overlap: a leading dimension is smaller than the row");
        const Rows xr{x, rows, K, ldx, 2}, qr{q, rows, K, K, 1}, sr{scale, 1, rows, rows, 4};
        CPM_REQUIRE(!overlap(xr, qr) && !overlap(xr, sr) && !overlap(qr, sr), "w8a8_quantize: x, q and scale must not overlap");
        require_device("w8a8_quantize");
        w8::RowSource src;
        src.x = static_cast<const bf16*>(x);
        src.ldx = ldx;
        w8::launch_quantize(src, rows, K, static_cast<int8_t*>(q), K, K, scale, nullptr, 0, stream_of(stream));
        return 0;
    });
}

long cpmcu_w8a8_workspace_bytes(int rows, int N, int K, int inter) {
    return guarded([&]() -> long {
        require_sizes("w8a8_workspace_bytes", rows, N, K);
        require_rows("w8a8_workspace_bytes", rows);
        CPM_REQUIRE(inter >= 0, "w8a8_workspace_bytes: inter must not be negative");
        if (inter > 0) {
            require_sizes("w8a8_workspace_bytes", rows, inter, K);
            require_sizes("w8a8_workspace_bytes", rows, N, inter);
        }
        return static_cast<long>(layout_of(rows, N, K, inter).total);
    });
}

int cpmcu_debug_w8a8_division(int rows, int N, int K, int gated, int32_t* out) {
    return guarded([&] {
        require_sizes("debug_w8a8_division", rows, N, K);
        require_rows("debug_w8a8_division", rows);
        CPM_REQUIRE(rows >= 2 && out != nullptr, "debug_w8a8_division: products of two rows and more are divided");
        require_device("debug_w8a8_division");
        int32_t d[6];
        w8::product_division(rows, N, K, gated != 0, d);
        std::copy(d, d + 6, out);
        return 0;
    });
}

int cpmcu_w8a8_linear(const void* x, long long ldx, const void* packed, const void* bias, const void* norm, float eps, const void* delta,
                      float delta_scale, void* total, void* y, long long ldy, int rows, int N, int K, void* workspace, long long workspace_bytes, void* stream) {
    return guarded([&] {
        require_sizes("w8a8_linear", rows, N, K);
        require_rows("w8a8_linear", rows);
        if (rows == 0) return 0;
        require_packed("w8a8_linear", packed);
        const w8::RowSource src = source_of("w8a8_linear", x, ldx, norm, eps, delta, delta_scale, total, rows, K, y, ldy, N);
        const Rows xr{x, rows, K, ldx, 2}, yr{y, rows, N, ldy, 2}, dr{delta, rows, K, K, 2}, tr{total, rows, K, K, 2}, nr{norm, 1, K, K, 2}, br{bias, 1, N, N, 2};
        const Rows pr = whole(packed, w8::packed_bytes(N, K, false));
        require_apart("w8a8_linear", {yr, tr}, {pr, br});
        const Layout l = layout_of(rows, N, K, 0);
        require_workspace("w8a8_linear", workspace, workspace_bytes, l, {xr, yr, dr, tr, nr, br, pr});
        require_device("w8a8_linear");
        cudaStream_t s = stream_of(stream);
        const w8::Packed w = w8::packed_view(packed, N, K, false);
        if (rows == 1) {
            w8::launch_one_row(src, N, K, w, static_cast<const bf16*>(bias), static_cast<bf16*>(y), nullptr, s);
            return 0;
        }
        char* ws = static_cast<char*>(workspace);
        w8::Product p;
        p.M = rows; p.N = N; p.K = K;
        p.w = w;
        int8_t* q = reinterpret_cast<int8_t*>(ws + l.q);
        float* xs = reinterpret_cast<float*>(ws + l.xs);
        p.q = q; p.xs = xs;
        p.bias = static_cast<const bf16*>(bias);
        p.y = static_cast<bf16*>(y); p.ldy = ldy;
        p.partials = ws + l.partials;
        p.tickets = reinterpret_cast<int*>(ws + l.tickets);
        w8::launch_quantize(src, rows, K, q, w8::pad_cols(K), w8::pad_cols(K), xs, p.tickets, l.n_tickets, s);
        w8::launch_product(p, s);
        return 0;
    });
}

int cpmcu_w8a8_ffn(const void* x, long long ldx, const void* gate_up, const void* down, const void* norm, float eps, const void* delta,
                   float delta_scale, void* total, void* y, long long ldy, int rows, int K, int inter, void* workspace, long long workspace_bytes, void* stream) {
    return guarded([&] {
        require_sizes("w8a8_ffn", rows, inter, K);
        require_sizes("w8a8_ffn", rows, K, inter);
        require_rows("w8a8_ffn", rows);
        if (rows == 0) return 0;
        require_packed("w8a8_ffn", gate_up);
        require_packed("w8a8_ffn", down);
        const w8::RowSource src = source_of("w8a8_ffn", x, ldx, norm, eps, delta, delta_scale, total, rows, K, y, ldy, K);
        const Rows xr{x, rows, K, ldx, 2}, yr{y, rows, K, ldy, 2}, dr{delta, rows, K, K, 2}, tr{total, rows, K, K, 2}, nr{norm, 1, K, K, 2};
        const Rows gr = whole(gate_up, w8::packed_bytes(inter, K, true)), pr = whole(down, w8::packed_bytes(K, inter, false));
        require_apart("w8a8_ffn", {yr, tr}, {gr, pr});
        const Layout l = layout_of(rows, K, K, inter);
        require_workspace("w8a8_ffn", workspace, workspace_bytes, l, {xr, yr, dr, tr, nr, gr, pr});
        require_device("w8a8_ffn");
        cudaStream_t s = stream_of(stream);
        const w8::Packed wg = w8::packed_view(gate_up, inter, K, true), wd = w8::packed_view(down, K, inter, false);
        char* ws = static_cast<char*>(workspace);
        float* act = reinterpret_cast<float*>(ws + l.act);
        // Activations in rows of a multiple of eight: the columns behind `inter` are products with the packed zeros, 0, or NaN in a row that is NaN anyway.
        const int middle_cols = static_cast<int>(l.act_ld);
        w8::RowSource middle;
        middle.x32 = act;
        middle.ldx = l.act_ld;
        if (rows == 1) {
            w8::launch_one_row(src, middle_cols, K, wg, nullptr, nullptr, act, s);
            w8::launch_one_row(middle, K, middle_cols, wd, nullptr, static_cast<bf16*>(y), nullptr, s);
            return 0;
        }
        int8_t* q = reinterpret_cast<int8_t*>(ws + l.q);
        float* xs = reinterpret_cast<float*>(ws + l.xs);
        w8::Product p;
        p.M = rows; p.N = middle_cols; p.K = K;
        p.w = wg;
        p.q = q; p.xs = xs;
        p.act = act; p.ldy = l.act_ld;
        w8::launch_quantize(src, rows, K, q, w8::pad_cols(K), w8::pad_cols(K), xs, nullptr, 0, s);
        w8::launch_product(p, s);
        p = w8::Product();
        p.M = rows; p.N = K; p.K = inter;
        p.w = wd;
        p.q = q; p.xs = xs;
        p.y = static_cast<bf16*>(y); p.ldy = ldy;
        p.partials = ws + l.partials;
        p.tickets = reinterpret_cast<int*>(ws + l.tickets);
        w8::launch_quantize(middle, rows, middle_cols, q, w8::pad_cols(inter), w8::pad_cols(inter), xs, p.tickets, l.n_tickets, s);
        w8::launch_product(p, s);
        return 0;
    });
}

int cpmcu_rotary_append(const void* qkv, long long ld, int rows, int heads, int kv_heads, int dim, int rot_dims, int interleaved, const float* inv_freq,
                        float factor, const int32_t* pos, void* q, long long ldq, void* k_cache, void* v_cache, int cache_rows, const int32_t* slots,
                        void* stream) {
    return guarded([&] {
        CPM_REQUIRE(rows >= 0 && heads >= 0 && kv_heads >= 0 && heads + kv_heads >= 1 && dim >= 2 && dim % 2 == 0,
                    "rotary_append: sizes must be positive and head widths even");
        CPM_REQUIRE(heads <= 65536 && kv_heads <= 65536 && dim <= 4096 && (static_cast<long long>(heads) + 2 * kv_heads) * dim < (1ll << 28), "rotary_append: rows are too wide");
        CPM_REQUIRE(rot_dims >= 0 && rot_dims <= dim && rot_dims % 2 == 0, "rotary_append: rot_dims is even and at most the head's width");
        CPM_REQUIRE(rot_dims / 2 <= rotary_max_pairs(), "rotary_append: at most 512 pairs are rotated");
        if (rows == 0) return 0;
        const long long kv_dim = static_cast<long long>(kv_heads) * dim, q_cols = static_cast<long long>(heads) * dim, cols = q_cols + 2 * kv_dim;
        CPM_REQUIRE(qkv != nullptr && pos != nullptr && (rot_dims == 0 || inv_freq != nullptr), "rotary_append: qkv, pos and inv_freq must not be null");
        CPM_REQUIRE(ld >= cols && (heads == 0 || ldq >= q_cols), "rotary_append: rows overlap: a leading dimension is smaller than the row");
        CPM_REQUIRE(heads == 0 || q != nullptr, "rotary_append: q must not be null");
        const Rows in{qkv, rows, cols, ld, 2}, qr{heads > 0 ? q : nullptr, rows, q_cols, ldq, 2};
        CPM_REQUIRE((q == qkv && (ldq == ld || rows == 1)) || !overlap(in, qr), "rotary_append: q must be the query part of qkv itself, or apart from it");
        if (kv_heads > 0) {
            CPM_REQUIRE(k_cache != nullptr && v_cache != nullptr && slots != nullptr && cache_rows >= 0, "rotary_append: caches and slots must not be null");
            const Rows kr{k_cache, cache_rows, kv_dim, kv_dim, 2}, vr{v_cache, cache_rows, kv_dim, kv_dim, 2};
            CPM_REQUIRE(!overlap(in, kr) && !overlap(in, vr) && !overlap(qr, kr) && !overlap(qr, vr) && !overlap(kr, vr),
                        "rotary_append: the caches must not overlap each other, qkv or q");
        }
        const Rows written[] = {qr, {kv_heads > 0 ? k_cache : nullptr, cache_rows, kv_dim, kv_dim, 2}, {kv_heads > 0 ? v_cache : nullptr, cache_rows, kv_dim, kv_dim, 2}};
        for (const Rows& w : written) {
            CPM_REQUIRE(!overlap(w, whole(pos, 4ull * rows)) && !overlap(w, whole(kv_heads > 0 ? slots : nullptr, 4ull * rows)) && !overlap(w, whole(inv_freq, 2ull * rot_dims)),
                        "rotary_append: q and the caches must not overlap positions, slots or frequencies");
        }
        require_device("rotary_append");
        RotaryArgs a;
        a.qkv = static_cast<const bf16*>(qkv);
        a.ld = ld;
        a.heads = heads; a.kv_heads = kv_heads; a.dim = dim; a.half = rot_dims / 2;
        a.inv_freq = inv_freq; a.factor = factor; a.pos = pos;
        a.q = static_cast<bf16*>(q);
        a.ldq = heads > 0 ? ldq : 0;
        a.k_cache = static_cast<bf16*>(k_cache); a.v_cache = static_cast<bf16*>(v_cache);
        a.cache_rows = cache_rows; a.slots = slots;
        a.errors = op_counters(stream_of(stream));
        launch_rotary(a, rows, interleaved != 0, stream_of(stream));
        return 0;
    });
}

}  // extern "C"
