// extern "C" surface declared in include/lancelot_b200.h.  Argument validation lives here
// (the kernels trust their launchers); nothing below ever computes on the CPU.
#include <algorithm>
#include <cstring>
#include <vector>

#include "context.h"

namespace lb {
const std::string &last_error();
int context_create(int logN, const std::vector<u64> &moduli, int size_P, const std::vector<uint32_t> &elts, int device,
                   Context **out);
void context_destroy(Context *ctx);
} // namespace lb

using namespace lb;

struct lb_context {
    Context *c;
};

static inline Context *C(lb_context *h) { return h ? h->c : nullptr; }
namespace lb {
Context *lb_context_impl(lb_context *h) { return h ? h->c : nullptr; }
} // namespace lb
static inline const Context *C(const lb_context *h) { return h ? h->c : nullptr; }
static inline cudaStream_t S(void *s) { return reinterpret_cast<cudaStream_t>(s); }

#define REQUIRE(cond, msg)             \
    do {                               \
        if (!(cond)) {                 \
            set_error(msg);            \
            return LB_ERR_INVALID_ARG; \
        }                              \
    } while (0)

static int bind(lb_context *h)
{
    if (!h || !h->c) {
        set_error("context is null");
        return LB_ERR_INVALID_ARG;
    }
    LB_CUDA(cudaSetDevice(h->c->device));
    return LB_OK;
}

static int level_ok(const Context *c, int size_l)
{
    REQUIRE(size_l >= 1 && size_l <= c->hp.size_Q, "size_l is out of range for this context");
    return LB_OK;
}

extern "C" {

const char *lb_last_error(void) { return last_error().c_str(); }

int lb_coeff_modulus_create(uint64_t n, const int *bit_sizes, int count, uint64_t *out)
{
    REQUIRE(bit_sizes && out && count >= 1 && count <= 64, "bit_sizes is invalid");
    REQUIRE(n >= 16 && n <= 131072 && (n & (n - 1)) == 0, "poly_modulus_degree is invalid");
    std::vector<int> bits(bit_sizes, bit_sizes + count);
    for (int b : bits) REQUIRE(b >= 2 && b <= 60, "bit_sizes is invalid");
    std::vector<u64> m = coeff_modulus_create(n, bits);
    if (m.empty()) {
        set_error("failed to find enough qualifying primes");
        return LB_ERR_LOGIC;
    }
    std::memcpy(out, m.data(), sizeof(u64) * count);
    return LB_OK;
}

int lb_galois_elts_from_steps(const int *steps, int count, uint64_t n, uint32_t *out)
{
    REQUIRE(steps && out && count >= 0, "steps is invalid");
    for (int i = 0; i < count; ++i) {
        const long a = steps[i] < 0 ? -(long)steps[i] : steps[i];
        REQUIRE(a < (long)(n >> 1), "step count too large");
        out[i] = galois_elt_from_step(steps[i], n);
    }
    return LB_OK;
}

uint64_t lb_minimal_primitive_root(uint64_t degree, uint64_t modulus) { return minimal_primitive_root(degree, modulus); }

int lb_max_bit_count_tc128(uint64_t n) { return max_bit_count_tc128(n); }

int lb_context_create(int log_n, const uint64_t *moduli, int n_moduli, int special, const uint32_t *elts, int n_elts,
                      int check_tc128, int device, lb_context **out)
{
    REQUIRE(out, "out is null");
    *out = nullptr;
    REQUIRE(moduli && n_moduli >= 1 && n_moduli <= 64, "coeff_modulus size is invalid");
    REQUIRE(n_elts >= 0 && (n_elts == 0 || elts), "galois_elts is invalid");
    std::vector<u64> m(moduli, moduli + n_moduli);
    std::vector<uint32_t> e(elts, elts + n_elts);
    if (check_tc128) {
        int bits = 0;
        for (u64 v : m) bits += 64 - __builtin_clzll(v);
        const int bound = max_bit_count_tc128(u64(1) << log_n);
        REQUIRE(bound > 0 && bits <= bound, "invalid parameters_insecure");
    }
    Context *c = nullptr;
    int rc = context_create(log_n, m, special, e, device, &c);
    if (rc) return rc;
    *out = new lb_context{c};
    return LB_OK;
}

void lb_context_destroy(lb_context *h)
{
    if (!h) return;
    context_destroy(h->c);
    delete h;
}

int lb_context_get_modulus(const lb_context *h, int i, uint64_t *out)
{
    const Context *c = C(h);
    REQUIRE(c && out && i >= 0 && i < c->hp.size_QP, "modulus index is out of range");
    *out = c->hp.q[i];
    return LB_OK;
}

int lb_context_get_root(const lb_context *h, int i, uint64_t *out)
{
    const Context *c = C(h);
    REQUIRE(c && out && i >= 0 && i < c->hp.size_QP, "modulus index is out of range");
    *out = c->hp.psi[i];
    return LB_OK;
}

int lb_context_get_galois_table(const lb_context *h, int e, uint32_t *out)
{
    const Context *c = C(h);
    REQUIRE(c && out && e >= 0 && e < (int)c->hp.galois_elts.size(), "Galois element index is out of range");
    std::memcpy(out, &c->hp.perm[(size_t)e * c->hp.N], c->hp.N * sizeof(uint32_t));
    return LB_OK;
}

int lb_context_reserve_workspace(lb_context *h, size_t bytes)
{
    int rc = bind(h);
    if (rc) return rc;
    return C(h)->ensure_workspace(bytes);
}

size_t lb_keyswitch_workspace_bytes(const lb_context *h, int size_l)
{
    const Context *c = C(h);
    if (!c || size_l < 1 || size_l > c->hp.size_Q || c->hp.size_P < 1) return 0;
    return keyswitch_workspace_bytes(c, size_l);
}

static int ntt_rows(lb_context *h, uint64_t *data, int n_groups, int size_l, int size_p, bool fwd, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    Context *c = C(h);
    REQUIRE(data || n_groups == 0, "data is null");
    REQUIRE(n_groups >= 0 && size_l >= 0 && size_l <= c->hp.size_Q && size_p >= 0 && size_p <= c->hp.size_P && size_l + size_p >= 1,
            "limb counts are out of range for this context");
    NttJob job;
    job.src = data;
    job.dst = data;
    job.n_groups = n_groups;
    job.per_group = size_l + size_p;
    job.size_l = size_l;
    return fwd ? ntt_forward(c, job, S(stream)) : ntt_inverse(c, job, S(stream));
}

int lb_ntt_forward(lb_context *h, uint64_t *data, int n_groups, int size_l, int size_p, void *stream)
{
    return ntt_rows(h, data, n_groups, size_l, size_p, true, stream);
}

int lb_ntt_inverse(lb_context *h, uint64_t *data, int n_groups, int size_l, int size_p, void *stream)
{
    return ntt_rows(h, data, n_groups, size_l, size_p, false, stream);
}

static int binary(lb_context *h, int op, int size_l, int n_polys, const uint64_t *a, const uint64_t *b, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(n_polys >= 0 && a && out && (b || op == OP_NEG || op == OP_REDUCE), "operand is null");
    return poly_binary(C(h), op, size_l, (long)n_polys * size_l, a, b, out, S(stream));
}

int lb_add(lb_context *h, int size_l, int n, const uint64_t *a, const uint64_t *b, uint64_t *out, void *s) { return binary(h, OP_ADD, size_l, n, a, b, out, s); }
int lb_sub(lb_context *h, int size_l, int n, const uint64_t *a, const uint64_t *b, uint64_t *out, void *s) { return binary(h, OP_SUB, size_l, n, a, b, out, s); }
int lb_multiply_poly(lb_context *h, int size_l, int n, const uint64_t *a, const uint64_t *b, uint64_t *out, void *s) { return binary(h, OP_MUL, size_l, n, a, b, out, s); }
int lb_negate(lb_context *h, int size_l, int n, const uint64_t *a, uint64_t *out, void *s) { return binary(h, OP_NEG, size_l, n, a, nullptr, out, s); }
int lb_reduce_mod(lb_context *h, int size_l, int n, const uint64_t *a, uint64_t *out, void *s) { return binary(h, OP_REDUCE, size_l, n, a, nullptr, out, s); }

int lb_sum_groups(lb_context *h, int size_l, int n_polys, int n_groups, const int *offsets, const int *indices, int n_items,
                  const uint64_t *in, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(offsets && in && out && n_polys >= 1 && n_groups >= 0, "operand is null");
    if (n_groups == 0) return LB_OK;
    REQUIRE(n_groups <= 65535, "too many groups");
    REQUIRE(offsets[0] == 0, "offsets must start at 0");
    for (int g = 0; g < n_groups; ++g) REQUIRE(offsets[g + 1] >= offsets[g], "offsets must not decrease");
    REQUIRE(offsets[n_groups] == 0 || indices, "operand is null");
    for (int t = 0; t < offsets[n_groups]; ++t) REQUIRE(indices[t] >= 0 && indices[t] < n_items, "item index is out of range");
    return poly_sum_groups(C(h), size_l, (long)n_polys * size_l, n_groups, offsets, indices, in, out, S(stream));
}

int lb_multiply_poly_key_level(lb_context *h, const uint64_t *a, const uint64_t *b, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(a && b && out, "operand is null");
    // at the key level the limb list is Q || P, which is also the table order
    return poly_binary(C(h), OP_MUL, C(h)->hp.size_QP, C(h)->hp.size_QP, a, b, out, S(stream));
}

int lb_multiply(lb_context *h, int size_l, int batch, const uint64_t *a, const uint64_t *b, uint64_t *out3, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(a && b && out3 && batch >= 0, "operand is null");
    REQUIRE(out3 != a && out3 != b, "the size-3 result cannot alias an input");
    return poly_tensor(C(h), size_l, batch, a, b, out3, S(stream));
}

int lb_square(lb_context *h, int size_l, int batch, const uint64_t *a, uint64_t *out3, void *stream)
{
    return lb_multiply(h, size_l, batch, a, a, out3, stream);
}

int lb_mod_switch_drop(lb_context *h, int size_l, int n_polys, const uint64_t *in, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(size_l >= 2 && size_l <= C(h)->hp.size_Q, "end of modulus switching chain reached");
    REQUIRE(in && out && n_polys >= 1, "operand is null");
    return poly_drop_last(C(h), size_l, n_polys, in, out, S(stream));
}

int lb_galois_permute(lb_context *h, int elt, int n_limbs, const uint64_t *in, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(in && out && in != out && n_limbs >= 0, "operand is null or aliased");
    return poly_galois(C(h), elt, n_limbs, in, out, S(stream));
}

int lb_modup(lb_context *h, int size_l, const uint64_t *cks, uint64_t *digits, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(cks && digits, "operand is null");
    return modup(C(h), size_l, cks, digits, S(stream));
}

int lb_keyswitch_inner_product(lb_context *h, int size_l, const uint64_t *digits, const uint64_t *evk, uint64_t *cx, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(digits && evk && cx, "operand is null");
    // digits carries its own limbs here, so the "own" source is the digit buffer itself:
    // pass a pointer the kernel never dereferences differently by materialising the rows
    Context *c = C(h);
    if ((rc = level_ok(c, size_l))) return rc;
    // own limbs of digit j sit at digits[j][j*alpha ..]; gather them into the workspace tail
    const HostParams &hp = c->hp;
    const int LP = size_l + hp.size_P, alpha = hp.size_P;
    REQUIRE(alpha >= 1, "key switching needs at least one special prime");
    if ((rc = c->ensure_workspace(keyswitch_workspace_bytes(c, size_l)))) return rc;
    u64 *own = reinterpret_cast<u64 *>(c->ws); // the coefficient scratch is free at this point
    for (int j = 0; j < hp.level[size_l].beta; ++j) {
        const int s = j * alpha, e = s + alpha < size_l ? s + alpha : size_l;
        LB_CUDA(cudaMemcpyAsync(own + (size_t)s * hp.N, digits + ((size_t)j * LP + s) * hp.N, (size_t)(e - s) * hp.N * 8,
                                cudaMemcpyDeviceToDevice, S(stream)));
    }
    return inner_product(c, size_l, digits, own, evk, cx, S(stream));
}

int lb_moddown(lb_context *h, int size_l, const uint64_t *cx, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(cx && out, "operand is null");
    return moddown(C(h), size_l, cx, out, S(stream));
}

int lb_keyswitch(lb_context *h, int size_l, uint64_t *ct, const uint64_t *cks, const uint64_t *evk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct && cks && evk, "operand is null");
    const size_t poly = (size_t)size_l * C(h)->hp.N;
    return keyswitch(C(h), size_l, cks, evk, ct, ct + poly, ct, S(stream));
}

int lb_relinearize(lb_context *h, int size_l, uint64_t *ct3, const uint64_t *rlk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct3 && rlk, "operand is null");
    return relinearize(C(h), size_l, 1, ct3, rlk, S(stream));
}

int lb_relinearize_batch(lb_context *h, int size_l, int batch, uint64_t *ct3, const uint64_t *rlk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct3 && rlk && batch >= 0, "operand is null");
    if (batch == 0) return LB_OK;
    return relinearize(C(h), size_l, batch, ct3, rlk, S(stream));
}

int lb_rescale(lb_context *h, int size_l, int n_polys, const uint64_t *in, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(in && out && n_polys >= 1, "operand is null");
    return rescale(C(h), size_l, n_polys, 1, in, size_l, out, S(stream));
}

int lb_rescale_strided(lb_context *h, int size_l, int batch, int polys_per_ct, const uint64_t *in, size_t ct_stride, uint64_t *out,
                       void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(in && out && batch >= 0 && polys_per_ct >= 1, "operand is null");
    REQUIRE(ct_stride % C(h)->hp.N == 0, "ciphertext stride must be a whole number of limbs");
    if (batch == 0) return LB_OK;
    return rescale(C(h), size_l, batch, polys_per_ct, in, (long)(ct_stride / C(h)->hp.N), out, S(stream));
}

int lb_rescale_no_alloc(lb_context *h, int size_l, int n_polys, const uint64_t *in, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(in && out, "operand is null");
    return rescale_static(C(h), size_l, n_polys, in, out, S(stream));
}

size_t lb_rescale_no_alloc_max_words(void) { return rescale_static_max_words(); }

int lb_rotate(lb_context *h, int size_l, uint64_t *ct, int elt, const uint64_t *glk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct && glk, "operand is null");
    return rotate(C(h), size_l, 1, ct, elt, glk, S(stream));
}

int lb_rotate_batch(lb_context *h, int size_l, int batch, uint64_t *ct, int elt, const uint64_t *glk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct && glk && batch >= 0, "operand is null");
    if (batch == 0) return LB_OK;
    return rotate(C(h), size_l, batch, ct, elt, glk, S(stream));
}

int lb_hoisting(lb_context *h, int size_l, uint64_t *ct, int n_steps, const int *elts, const uint64_t *const *keys, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct && elts && keys, "operand is null");
    return hoisting(C(h), size_l, 1, ct, n_steps, elts, keys, S(stream));
}

int lb_hoisting_batch(lb_context *h, int size_l, int batch, uint64_t *ct, int n_steps, const int *elts, const uint64_t *const *keys,
                      void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(ct && elts && keys && batch >= 0, "operand is null");
    if (batch == 0) return LB_OK;
    return hoisting(C(h), size_l, batch, ct, n_steps, elts, keys, S(stream));
}

int lb_krum_accumulate(lb_context *h, int size_l, int n_chunks, const uint64_t *a, const uint64_t *b, size_t sa, size_t sb,
                       uint64_t *acc, int accumulate, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(a && b && acc && n_chunks >= 0, "operand is null");
    REQUIRE(sa % 2 == 0 && sb % 2 == 0, "chunk strides must be even");
    return krum_accumulate(C(h), size_l, n_chunks, a, b, (long)sa, (long)sb, acc, accumulate, S(stream));
}

int lb_krum_accumulate_tile(lb_context *h, int size_l, int n_chunks, int n_a, const uint64_t *const *a, int n_b,
                            const uint64_t *const *b, size_t chunk_stride, uint64_t *const *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(a && out && (b || n_b == 0) && n_chunks >= 0, "operand is null");
    REQUIRE(n_a >= 1 && n_a <= 4 && n_b >= 0 && n_b <= 4, "tile shape is out of range");
    for (int i = 0; i < n_a; ++i) REQUIRE(a[i], "operand is null");
    for (int i = 0; i < n_b; ++i) REQUIRE(b[i], "operand is null");
    const int n_pairs = n_b ? n_a * n_b : n_a * (n_a - 1) / 2;
    for (int i = 0; i < n_pairs && i < 8; ++i) REQUIRE(out[i], "operand is null");
    return krum_accumulate_tile(C(h), size_l, n_chunks, n_a, a, n_b, b, (long)chunk_stride, out, S(stream));
}

// The pair list of a round as tiles of lb_krum_accumulate_tile.  Clients are blocked by index in groups of four; a
// diagonal block whose pairs are all the pairs of its clients is one triangle, anything else is cut into rectangles of
// one or two first clients that share their set of second clients.
int lb_krum_pair_sums(lb_context *h, int size_l, int n_clients, const uint64_t *const *cts, int n_chunks, size_t chunk_stride,
                      int n_pairs, const int *pairs, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(cts && out && (pairs || n_pairs == 0) && n_chunks >= 0 && n_pairs >= 0 && n_clients >= 0, "operand is null");
    for (int p = 0; p < n_pairs; ++p) {
        const int i = pairs[2 * p], j = pairs[2 * p + 1];
        REQUIRE(i >= 0 && i < j && j < n_clients, "a pair is (i, j) with 0 <= i < j < n_clients");
        REQUIRE(cts[i] && cts[j], "operand is null");
    }
    constexpr int W = 4;
    const size_t acc_words = (size_t)3 * size_l * C(h)->hp.N;
    const int n_blocks = (n_clients + W - 1) / W;
    // slot[i * n_clients + j] = index of pair (i, j) in the caller's list, -1 if absent (a pair listed twice is refused)
    std::vector<int> slot((size_t)n_clients * n_clients, -1);
    for (int p = 0; p < n_pairs; ++p) {
        int &sl = slot[(size_t)pairs[2 * p] * n_clients + pairs[2 * p + 1]];
        REQUIRE(sl < 0, "a pair is listed twice");
        sl = p;
    }
    auto launch = [&](const std::vector<int> &rows, const std::vector<int> &cols) -> int {
        const uint64_t *a[4], *b[4];
        uint64_t *o[8];
        const int na = (int)rows.size(), nb = (int)cols.size();
        for (int r = 0; r < na; ++r) a[r] = cts[rows[r]];
        for (int c = 0; c < nb; ++c) b[c] = cts[cols[c]];
        int n = 0;
        if (nb == 0) {
            for (int r = 0; r < na; ++r)
                for (int c = r + 1; c < na; ++c) o[n++] = out + (size_t)slot[(size_t)rows[r] * n_clients + rows[c]] * acc_words;
        } else {
            for (int r = 0; r < na; ++r)
                for (int c = 0; c < nb; ++c) o[n++] = out + (size_t)slot[(size_t)rows[r] * n_clients + cols[c]] * acc_words;
        }
        return krum_accumulate_tile(C(h), size_l, n_chunks, na, a, nb, nb ? b : nullptr, (long)chunk_stride, o, S(stream));
    };
    for (int ga = 0; ga < n_blocks; ++ga) {
        for (int gb = ga; gb < n_blocks; ++gb) {
            // the block's pairs by first client
            std::vector<int> first;
            std::vector<std::vector<int>> second;
            int count = 0;
            std::vector<char> seen(n_clients, 0);
            std::vector<int> members;
            for (int i = ga * W; i < (ga + 1) * W && i < n_clients; ++i) {
                std::vector<int> cols;
                for (int j = gb * W; j < (gb + 1) * W && j < n_clients; ++j)
                    if (j > i && slot[(size_t)i * n_clients + j] >= 0) {
                        cols.push_back(j);
                        if (!seen[i]) seen[i] = 1, members.push_back(i);
                        if (!seen[j]) seen[j] = 1, members.push_back(j);
                    }
                if (!cols.empty()) {
                    first.push_back(i);
                    count += (int)cols.size();
                    second.push_back(cols);
                }
            }
            if (count == 0) continue;
            const int m = (int)members.size();
            if (ga == gb && count == m * (m - 1) / 2) {
                std::sort(members.begin(), members.end());
                if ((rc = launch(members, {}))) return rc;
                continue;
            }
            for (size_t k = 0; k < first.size();) {
                if (k + 1 < first.size() && second[k + 1] == second[k]) {
                    if ((rc = launch({first[k], first[k + 1]}, second[k]))) return rc;
                    k += 2;
                } else {
                    if ((rc = launch({first[k]}, second[k]))) return rc;
                    k += 1;
                }
            }
        }
    }
    return LB_OK;
}

// byzantine_fl.py:244-273 for a batch of pair sums: relinearize_inplace, rescale_to_next_inplace, hoisting over
// the first steps added to the ciphertext, then rotate_vector + add_inplace for every further step
int lb_krum_scores(lb_context *h, int size_l, int n_pairs, uint64_t *acc, const uint64_t *relin_key, int n_first, const int *first_elts,
                   const uint64_t *const *first_keys, int n_pow, const int *pow_elts, const uint64_t *const *pow_keys, uint64_t *scores,
                   void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(size_l >= 2, "the pair sums must have a level to rescale to");
    REQUIRE(acc && relin_key && scores && n_pairs >= 0 && n_first >= 0 && n_pow >= 0, "operand is null");
    REQUIRE((n_first == 0 || (first_elts && first_keys)) && (n_pow == 0 || (pow_elts && pow_keys)), "operand is null");
    if (n_pairs == 0) return LB_OK;
    Context *c = C(h);
    cudaStream_t st = S(stream);
    const int L = size_l - 1;
    if ((rc = relinearize(c, size_l, n_pairs, acc, relin_key, st))) return rc;
    if ((rc = rescale(c, size_l, n_pairs, 2, acc, 3L * size_l, scores, st))) return rc;
    // scores += hoisting(scores), scores += rotate(scores, step): the sums are formed inside the key switch's closing
    // transform (no copy of the batch, no separate addition)
    if (n_first > 0 && (rc = hoisting(c, L, n_pairs, scores, n_first, first_elts, first_keys, st, true))) return rc;
    for (int k = 0; k < n_pow; ++k)
        if ((rc = rotate(c, L, n_pairs, scores, pow_elts[k], pow_keys[k], st, true))) return rc;
    return LB_OK;
}

int lb_decrypt(lb_context *h, int size_l, int n_polys, const uint64_t *ct, const uint64_t *sk, uint64_t *pt, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(ct && sk && pt && n_polys >= 1, "operand is null");
    return poly_decrypt(C(h), size_l, n_polys, 1, ct, sk, pt, S(stream));
}

int lb_decrypt_batch(lb_context *h, int size_l, int n_polys, int batch, const uint64_t *ct, const uint64_t *sk, uint64_t *pt, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(ct && sk && pt && n_polys >= 1 && batch >= 0, "operand is null");
    if (batch == 0) return LB_OK;
    return poly_decrypt(C(h), size_l, n_polys, batch, ct, sk, pt, S(stream));
}

int lb_mask_accumulate(lb_context *h, int size_l, int n_clients, int n_chunks, const uint64_t *const *client_cts, size_t chunk_stride,
                       const uint64_t *masks, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(client_cts && masks && out && n_chunks >= 0, "operand is null");
    REQUIRE(chunk_stride % 2 == 0, "chunk stride must be even");
    return mask_accumulate(C(h), size_l, n_clients, n_chunks, client_cts, (long)chunk_stride, masks, out, S(stream));
}

// ---- samplers, keys, encryption ------------------------------------------------------------

static int stage_seeds(Context *c, const uint8_t *host_seeds, int n_seeds, uint32_t **d_seeds, u64 **scratch, size_t scratch_words,
                       cudaStream_t stream)
{
    // layout of the context scratch: [seeds][scratch_words]
    const size_t seed_bytes = ((size_t)n_seeds * 64 + 255) / 256 * 256;
    int rc = c->ensure_workspace(seed_bytes + scratch_words * 8);
    if (rc) return rc;
    *d_seeds = reinterpret_cast<uint32_t *>(c->ws);
    if (scratch) *scratch = reinterpret_cast<u64 *>(reinterpret_cast<uint8_t *>(c->ws) + seed_bytes);
    LB_CUDA(cudaMemcpyAsync(*d_seeds, host_seeds, (size_t)n_seeds * 64, cudaMemcpyHostToDevice, stream));
    return LB_OK;
}

int lb_sample_ternary(lb_context *h, const uint8_t *seed, int size_l, int size_p, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(seed && out, "operand is null");
    uint32_t *ds;
    if ((rc = stage_seeds(C(h), seed, 1, &ds, nullptr, 0, S(stream)))) return rc;
    return sample_small(C(h), 0, ds, 16, 1, size_l, size_p, out, S(stream));
}

int lb_sample_error(lb_context *h, const uint8_t *seed, int size_l, int size_p, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(seed && out, "operand is null");
    uint32_t *ds;
    if ((rc = stage_seeds(C(h), seed, 1, &ds, nullptr, 0, S(stream)))) return rc;
    return sample_small(C(h), 1, ds, 16, 1, size_l, size_p, out, S(stream));
}

int lb_sample_uniform(lb_context *h, const uint8_t *seed, int size_l, int size_p, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(seed && out, "operand is null");
    REQUIRE(C(h)->hp.logN >= 3, "ring degree too small");
    uint32_t *ds;
    if ((rc = stage_seeds(C(h), seed, 1, &ds, nullptr, 0, S(stream)))) return rc;
    return sample_uniform(C(h), ds, 16, 1, size_l, size_p, out, S(stream));
}

int lb_gen_secret_key(lb_context *h, const uint8_t *seed, uint64_t *sk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(seed && sk, "operand is null");
    Context *c = C(h);
    uint32_t *ds;
    if ((rc = stage_seeds(c, seed, 1, &ds, nullptr, 0, S(stream)))) return rc;
    if ((rc = sample_small(c, 0, ds, 16, 1, c->hp.size_Q, c->hp.size_P, sk, S(stream)))) return rc;
    NttJob j;
    j.src = sk;
    j.dst = sk;
    j.n_groups = 1;
    j.per_group = c->hp.size_QP;
    j.size_l = c->hp.size_Q;
    return ntt_forward(c, j, S(stream));
}

int lb_gen_public_key(lb_context *h, const uint64_t *sk, const uint8_t *seed_error, const uint8_t *seed_uniform, uint64_t *pk, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(sk && seed_error && seed_uniform && pk, "operand is null");
    Context *c = C(h);
    uint8_t both[128];
    memcpy(both, seed_error, 64);
    memcpy(both + 64, seed_uniform, 64);
    uint32_t *ds;
    u64 *scratch;
    if ((rc = stage_seeds(c, both, 2, &ds, &scratch, (size_t)c->hp.size_QP << c->hp.logN, S(stream)))) return rc;
    // the staged copy must not be overwritten by `both` going out of scope: pageable copies complete before return
    return gen_public_key(c, sk, ds, ds + 16, pk, scratch, S(stream));
}

int lb_gen_switch_key(lb_context *h, const uint64_t *sk, const uint64_t *sk_target, const uint8_t *seeds, uint64_t *out, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(sk && sk_target && seeds && out, "operand is null");
    Context *c = C(h);
    REQUIRE(c->hp.size_P >= 1 && c->hp.size_Q % c->hp.size_P == 0, "special_modulus_size must divide the number of data primes");
    const int dnum = c->hp.size_Q / c->hp.size_P;
    uint32_t *ds;
    u64 *scratch;
    if ((rc = stage_seeds(c, seeds, 2 * dnum, &ds, &scratch, (size_t)c->hp.size_QP << c->hp.logN, S(stream)))) return rc;
    return gen_switch_key(c, sk, sk_target, ds, out, scratch, S(stream));
}

int lb_gen_galois_keys(lb_context *h, const uint64_t *sk, int n_keys, const int *elt_indices, const uint8_t *seeds, uint64_t *out,
                       void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(sk && seeds && out && n_keys >= 0 && (elt_indices || n_keys == 0), "operand is null");
    if (n_keys == 0) return LB_OK;
    Context *c = C(h);
    REQUIRE(c->hp.size_P >= 1 && c->hp.size_Q % c->hp.size_P == 0, "special_modulus_size must divide the number of data primes");
    for (int k = 0; k < n_keys; ++k)
        REQUIRE(elt_indices[k] >= 0 && elt_indices[k] < (int)c->hp.galois_elts.size(), "Galois element index is out of range");
    const int dnum = c->hp.size_Q / c->hp.size_P;
    const size_t poly = (size_t)c->hp.size_QP << c->hp.logN;
    uint32_t *ds;
    u64 *scratch;
    // scratch: the rotated secret keys [n][QP][N], then one error polynomial per key and digit, then the same as signed bytes
    const size_t errors8 = ((size_t)n_keys * dnum * c->hp.N + 7) / 8;
    if ((rc = stage_seeds(c, seeds, 2 * dnum * n_keys, &ds, &scratch, poly * (size_t)n_keys * (1 + dnum) + errors8, S(stream)))) return rc;
    u64 *targets = scratch, *errors = scratch + poly * n_keys;
    if ((rc = poly_galois_many(c, elt_indices, n_keys, c->hp.size_QP, sk, targets, S(stream)))) return rc;
    return gen_switch_keys(c, sk, targets, n_keys, ds, out, errors, S(stream));
}

int lb_encrypt_asymmetric(lb_context *h, const uint64_t *pk, const uint64_t *pt, const uint8_t *seeds, int batch, uint64_t *ct, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(pk && seeds && ct && batch >= 0, "operand is null");
    if (batch == 0) return LB_OK;
    return encrypt_asymmetric(C(h), pk, pt, 0, seeds, batch, ct, S(stream));
}

int lb_encode_encrypt(lb_context *h, const uint64_t *pk, const void *values, int dtype, size_t value_stride, int n_values,
                      int sparse_slots, int batch, double scale, const uint8_t *seeds, uint64_t *ct, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(pk && seeds && ct && batch >= 0 && (values || n_values == 0), "operand is null");
    REQUIRE(dtype >= 0 && dtype <= 2, "unknown value type");
    if (batch == 0) return LB_OK;
    Context *c = C(h);
    const int Q = c->hp.size_Q;
    // coefficient-form plaintexts live behind the encryption scratch
    const size_t enc_bytes = (encrypt_workspace_bytes(c, batch) + 255) / 256 * 256;
    const size_t pt_bytes = ((size_t)batch * Q << c->hp.logN) * 8;
    if ((rc = c->ensure_workspace(enc_bytes + pt_bytes))) return rc;
    u64 *pt = reinterpret_cast<u64 *>(reinterpret_cast<uint8_t *>(c->ws) + enc_bytes);
    // the encryption's scratch (its first rows hold N / 2 complex values per message) is free while the messages are encoded
    if ((rc = encode(c, Q, values, dtype, (long)value_stride, n_values, sparse_slots, batch, scale, pt, c->d_status, 1, S(stream),
                     reinterpret_cast<double *>(c->ws))))
        return rc;
    return encrypt_asymmetric(c, pk, pt, 1, seeds, batch, ct, S(stream));
}

// ---- encoder ------------------------------------------------------------------------------

int lb_encode(lb_context *h, int size_l, const void *values, int dtype, size_t value_stride, int n_values, int sparse_slots, int batch,
              double scale, uint64_t *pt, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE((values || n_values == 0) && pt && batch >= 0 && n_values >= 0, "values cannot be null");
    REQUIRE(dtype >= 0 && dtype <= 2, "unknown value type");
    return encode(C(h), size_l, values, dtype, (long)value_stride, n_values, sparse_slots, batch, scale, pt, C(h)->d_status, 0, S(stream));
}

int lb_decode(lb_context *h, int size_l, const uint64_t *pt, double scale, int sparse_slots, double *out_complex, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(pt && out_complex, "destination cannot be null");
    return decode(C(h), size_l, 1, pt, scale, sparse_slots, out_complex, S(stream));
}

int lb_decode_batch(lb_context *h, int size_l, int batch, const uint64_t *pt, double scale, int sparse_slots, double *out_complex, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = level_ok(C(h), size_l))) return rc;
    REQUIRE(pt && out_complex && batch >= 0, "destination cannot be null");
    if (batch == 0) return LB_OK;
    return decode(C(h), size_l, batch, pt, scale, sparse_slots, out_complex, S(stream));
}

// ---- 8-bit updates ---------------------------------------------------------------------------

static int cache_ok(const int8_t *codes, int64_t code_stride, const float *scales, int64_t scale_stride, int64_t n_slots, int64_t page,
                    int64_t group)
{
    REQUIRE(page >= 16 && page % 16 == 0 && page <= (1 << 30), "a page holds a multiple of 16 codes, at most 2^30");
    REQUIRE(group == 0 || (group >= 32 && group <= (1 << 30) && (group & (group - 1)) == 0), "group is 0 or a power of two from 32 on");
    REQUIRE(n_slots >= 0 && n_slots < (int64_t)1 << 31, "n_slots is out of range");
    REQUIRE(n_slots == 0 || (codes && scales), "operand is null");
    REQUIRE((uintptr_t)codes % 16 == 0 && code_stride % 16 == 0 && code_stride >= page, "the slots of a cache start on 16-byte boundaries and do not overlap");
    const int64_t groups = group && group < page ? (page + group - 1) / group : 1;
    REQUIRE((uintptr_t)scales % 4 == 0 && scale_stride >= groups, "the scales of two slots overlap");
    return LB_OK;
}

static int value_size(int dtype) { return dtype == 1 ? 4 : dtype == 3 || dtype == 4 ? 2 : 0; }

// rows x cols of elements of `size` bytes at p, `stride` elements apart
static int rows_ok(const void *p, int64_t rows, int64_t cols, int64_t stride, int size)
{
    REQUIRE(p, "operand is null");
    REQUIRE((uintptr_t)p % size == 0, "an operand is not aligned to its type");
    REQUIRE(rows <= 1 || (stride >= cols && stride <= (int64_t)1 << 40), "the rows of an operand overlap");
    return LB_OK;
}

// whether two operands of the same shape and stride have no element in common: one lies behind the other, or the rows of one lie in the gaps
// of the other
static bool rows_apart(const float *x, const float *y, int64_t rows, int64_t cols, int64_t stride)
{
    const int64_t span = (rows - 1) * stride + cols, d = ((int64_t)(intptr_t)y - (int64_t)(intptr_t)x) / 4;
    if (d >= span || d <= -span) return true;
    if (rows == 1) return false;
    const int64_t in = d >= 0 ? d % stride : (stride - -d % stride) % stride; // of y's row in the room of a row of x
    return in >= cols && in + cols <= stride;
}

// warps that a call over `pages` pages launches at most: their number has to fit the grid's arithmetic
static int pages_ok(int64_t n_rows, int64_t n_cols, int64_t page)
{
    REQUIRE(n_rows >= 0 && n_cols >= 0 && n_rows <= ((int64_t)1 << 31) - 1 && n_cols <= (int64_t)1 << 40, "n_rows or n_cols is out of range");
    const int64_t pages = (n_cols + page - 1) / page, per_page = (page + 31) / 32;
    REQUIRE(pages == 0 || n_rows <= (((int64_t)1 << 31) - 1) / pages / per_page, "too many rows for one call");
    return LB_OK;
}

static int workspace_ok(const void *workspace, size_t have, size_t need)
{
    REQUIRE(have >= need && (need == 0 || workspace), "the workspace is too small");
    REQUIRE(need == 0 || (uintptr_t)workspace % 16 == 0, "the workspace is not on a 16-byte boundary");
    return LB_OK;
}

size_t lb_quantize_rows_workspace_bytes(int64_t n_rows, int64_t n_cols, int64_t page, int64_t group)
{
    if (page < 16 || page > (1 << 30) || n_rows < 1 || n_cols < 1 || group < 0) return 0;
    return quantize_workspace_bytes(n_rows, n_cols, (int)page, (int)(group > page ? page : group));
}

int lb_quantize_rows(lb_context *h, const void *values, int dtype, int64_t n_rows, int64_t n_cols, int64_t value_stride, const int32_t *lengths,
                     const float *residual, float *residual_out, int64_t residual_stride, const int32_t *slots, int64_t n_slots, int64_t page,
                     int64_t group, int8_t *codes, int64_t code_stride, float *scales, int64_t scale_stride, void *workspace,
                     size_t workspace_bytes, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    if ((rc = cache_ok(codes, code_stride, scales, scale_stride, n_slots, page, group))) return rc;
    if ((rc = pages_ok(n_rows, n_cols, page))) return rc;
    if (n_rows == 0 || n_cols == 0) return LB_OK;
    if ((rc = rows_ok(values, n_rows, n_cols, value_stride, value_size(dtype)))) return rc;
    if (residual && (rc = rows_ok(residual, n_rows, n_cols, residual_stride, 4))) return rc;
    if (residual_out && (rc = rows_ok(residual_out, n_rows, n_cols, residual_stride, 4))) return rc;
    REQUIRE(!residual || !residual_out || residual == residual_out || rows_apart(residual, residual_out, n_rows, n_cols, residual_stride),
            "residual_out is residual itself or apart from it");
    REQUIRE((uintptr_t)lengths % 4 == 0 && (uintptr_t)slots % 4 == 0, "an operand is not aligned to its type");
    REQUIRE(slots || n_rows * ((n_cols + page - 1) / page) <= n_slots, "the cache has too few slots");
    if ((rc = workspace_ok(workspace, workspace_bytes, lb_quantize_rows_workspace_bytes(n_rows, n_cols, page, group)))) return rc;
    return quantize_rows(values, dtype, n_rows, n_cols, value_stride, lengths, residual, residual_out, residual_stride, slots, n_slots, (int)page,
                         (int)(group > page ? page : group), reinterpret_cast<signed char *>(codes), code_stride, scales, scale_stride, workspace,
                         C(h)->d_status, S(stream));
}

int lb_dequantize_rows(lb_context *h, const int8_t *codes, int64_t code_stride, const float *scales, int64_t scale_stride, int64_t n_slots,
                       int64_t page, int64_t group, const int32_t *slots, int64_t n_rows, int64_t n_cols, void *out, int dtype,
                       int64_t out_stride, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    if ((rc = cache_ok(codes, code_stride, scales, scale_stride, n_slots, page, group))) return rc;
    if ((rc = pages_ok(n_rows, n_cols, page))) return rc;
    if (n_rows == 0 || n_cols == 0) return LB_OK;
    if ((rc = rows_ok(out, n_rows, n_cols, out_stride, value_size(dtype)))) return rc;
    REQUIRE((uintptr_t)slots % 4 == 0, "an operand is not aligned to its type");
    REQUIRE(slots || n_rows * ((n_cols + page - 1) / page) <= n_slots, "the cache has too few slots");
    return dequantize_rows(reinterpret_cast<const signed char *>(codes), code_stride, scales, scale_stride, n_slots, (int)page,
                           (int)(group > page ? 0 : group), slots, n_rows, n_cols, out, dtype, out_stride, S(stream));
}

size_t lb_int8_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, const int8_t *a, int64_t a_stride, const int8_t *b, int64_t b_stride)
{
    if (m < 1 || n < 1 || k < 0 || m > (1 << 30) || n > (1 << 30) || k > 131071) return 0;
    return int8_matmul_workspace_bytes((int)m, (int)n, (int)k, a, a_stride, b, b_stride);
}

int lb_int8_matmul(lb_context *h, int64_t m, int64_t n, int64_t k, const int8_t *a, int64_t a_stride, const float *a_scale, const int8_t *b,
                   int64_t b_stride, const float *b_scale, void *out, int dtype, int64_t out_stride, void *workspace, size_t workspace_bytes,
                   void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    REQUIRE(m >= 0 && n >= 0 && k >= 0 && m <= (1 << 30) && n <= (1 << 30), "m, n or k is out of range");
    REQUIRE(k <= 131071, "a sum of more than 131071 products of 8-bit integers may pass 32 bits");
    if (m == 0 || n == 0) return LB_OK;
    if ((rc = rows_ok(out, m, n, out_stride, value_size(dtype)))) return rc;
    if (k > 0 && ((rc = rows_ok(a, m, k, a_stride, 1)) || (rc = rows_ok(b, n, k, b_stride, 1)))) return rc;
    REQUIRE(a_scale && b_scale, "operand is null");
    REQUIRE((uintptr_t)a_scale % 4 == 0 && (uintptr_t)b_scale % 4 == 0, "an operand is not aligned to its type");
    if ((rc = workspace_ok(workspace, workspace_bytes, lb_int8_matmul_workspace_bytes(m, n, k, a, a_stride, b, b_stride)))) return rc;
    return int8_matmul(C(h), (int)m, (int)n, (int)k, reinterpret_cast<const signed char *>(a), a_stride, a_scale,
                       reinterpret_cast<const signed char *>(b), b_stride, b_scale, out, dtype, out_stride, workspace, S(stream));
}

size_t lb_int8_distances_workspace_bytes(const lb_context *h, int64_t n, int64_t n_pages, int64_t page)
{
    if (!h || !h->c || n < 1 || n > 4096 || n_pages < 0 || page < 16 || page > (1 << 30)) return 0;
    return int8_distances_workspace_bytes(h->c, (int)n, n_pages, (int)page);
}

int lb_int8_distances(lb_context *h, const int8_t *codes, int64_t code_stride, const float *scales, int64_t scale_stride, int64_t n_slots,
                      int64_t page, int64_t group, const int32_t *slots, int64_t n, int64_t n_pages, double *out, void *workspace,
                      size_t workspace_bytes, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    if ((rc = cache_ok(codes, code_stride, scales, scale_stride, n_slots, page, group))) return rc;
    REQUIRE(n >= 0 && n <= 4096, "n is at most 4096");
    REQUIRE(n_pages >= 0 && n_pages <= (((int64_t)1 << 31) - 1) / ((page + 127) / 128), "too many pages for one call");
    if (n == 0) return LB_OK;
    REQUIRE(n * n_pages < (int64_t)1 << 31 && code_stride < (int64_t)1 << 31 && scale_stride < (int64_t)1 << 31, "the cache is too large for one call");
    REQUIRE(out, "operand is null");
    REQUIRE((uintptr_t)out % 8 == 0 && (uintptr_t)slots % 4 == 0, "an operand is not aligned to its type");
    REQUIRE(slots || n * n_pages <= n_slots, "the cache has too few slots");
    if ((rc = workspace_ok(workspace, workspace_bytes, lb_int8_distances_workspace_bytes(h, n, n_pages, page)))) return rc;
    return int8_distances(C(h), reinterpret_cast<const signed char *>(codes), code_stride, scales, scale_stride, n_slots, (int)page,
                          (int)(group > page ? 0 : group), slots, (int)n, (int)n_pages, out, workspace, S(stream));
}

// ---- 8-bit floating point, clipping -----------------------------------------------------------------------

static int code_type_ok(int code_type)
{
    REQUIRE(code_type == 5 || code_type == 6, "code_type is 5 (e4m3) or 6 (e5m2)");
    return LB_OK;
}
static int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

int lb_quantize_fp8(lb_context *h, const void *values, int dtype, int64_t n_rows, int64_t n_cols, int64_t value_stride, int blocks, int code_type,
                    uint8_t *codes, int64_t code_stride, float *scales, int64_t scale_stride, uint8_t *codes_down, int64_t code_down_stride,
                    float *scales_down, int64_t scale_down_stride, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    REQUIRE(blocks >= 1 && blocks <= 4, "blocks is 1 (rows), 2 (columns), 3 (both) or 4 (square)");
    if ((rc = code_type_ok(code_type))) return rc;
    REQUIRE(n_rows >= 0 && n_cols >= 0 && n_rows <= (int64_t)1 << 31 && n_cols <= (1 << 30), "n_rows or n_cols is out of range");
    if (n_rows == 0 || n_cols == 0) return LB_OK;
    REQUIRE(blocks_of(n_rows) * blocks_of(n_cols) < (int64_t)1 << 31, "too many blocks for one call");
    if ((rc = rows_ok(values, n_rows, n_cols, value_stride, value_size(dtype)))) return rc;
    if (blocks != 2) {
        if ((rc = rows_ok(codes, n_rows, n_cols, code_stride, 1))) return rc;
        if ((rc = rows_ok(scales, blocks == 4 ? blocks_of(n_rows) : n_rows, blocks_of(n_cols), scale_stride, 4))) return rc;
    }
    if (blocks == 2 || blocks == 3) {
        if ((rc = rows_ok(codes_down, n_rows, n_cols, code_down_stride, 1))) return rc;
        if ((rc = rows_ok(scales_down, blocks_of(n_rows), n_cols, scale_down_stride, 4))) return rc;
    }
    return quantize_fp8(values, dtype, n_rows, (int)n_cols, value_stride, blocks, code_type, codes, code_stride, scales, scale_stride, codes_down,
                        code_down_stride, scales_down, scale_down_stride, S(stream));
}

int lb_dequantize_fp8(lb_context *h, const uint8_t *codes, int code_type, int64_t code_stride, const float *scales, int64_t scale_stride, int blocks,
                      int64_t n_rows, int64_t n_cols, void *out, int dtype, int64_t out_stride, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    REQUIRE(blocks == 1 || blocks == 2 || blocks == 4, "blocks is 1 (rows), 2 (columns) or 4 (square)");
    if ((rc = code_type_ok(code_type))) return rc;
    REQUIRE(n_rows >= 0 && n_cols >= 0 && n_rows <= (int64_t)1 << 31 && n_cols <= (1 << 30), "n_rows or n_cols is out of range");
    if (n_rows == 0 || n_cols == 0) return LB_OK;
    REQUIRE(blocks_of(n_rows) * blocks_of(n_cols) < (int64_t)1 << 31, "too many blocks for one call");
    if ((rc = rows_ok(codes, n_rows, n_cols, code_stride, 1))) return rc;
    if ((rc = rows_ok(scales, blocks == 1 ? n_rows : blocks_of(n_rows), blocks == 2 ? n_cols : blocks_of(n_cols), scale_stride, 4))) return rc;
    if ((rc = rows_ok(out, n_rows, n_cols, out_stride, value_size(dtype)))) return rc;
    return dequantize_fp8(codes, code_type, code_stride, scales, scale_stride, blocks, n_rows, (int)n_cols, out, dtype, out_stride, S(stream));
}

static Fp8Operand operand_of(const lb_fp8_operand *o)
{
    return Fp8Operand{o->codes, o->stride, o->across, o->code_type, o->scales, o->scale_row, o->scale_block, o->scale_rows == 128 ? 7 : 0};
}
static int operand_ok(const lb_fp8_operand *o, int64_t rows, int64_t k)
{
    REQUIRE(o, "operand is null");
    int rc = code_type_ok(o->code_type);
    if (rc) return rc;
    REQUIRE(o->across == 0 || o->across == 1, "across is 0 or 1");
    REQUIRE(o->scale_rows == 1 || o->scale_rows == 128, "a scale is for 1 row or for 128");
    if (k == 0 || rows == 0) return LB_OK;
    if ((rc = rows_ok(o->codes, o->across ? k : rows, o->across ? rows : k, o->stride, 1))) return rc;
    REQUIRE(o->scales && (uintptr_t)o->scales % 4 == 0, "the scales are null or not aligned to their type");
    const int64_t n = o->scale_rows == 128 ? blocks_of(rows) : rows;
    REQUIRE((n <= 1 || (o->scale_row >= 0 && o->scale_row <= (int64_t)1 << 40)) && (k <= 128 || (o->scale_block >= 0 && o->scale_block <= (int64_t)1 << 40)),
            "a stride of the scales is out of range");
    return LB_OK;
}

size_t lb_fp8_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, const lb_fp8_operand *a, const lb_fp8_operand *b)
{
    if (m < 1 || n < 1 || k < 1 || m > (1 << 30) || n > (1 << 30) || k > (1 << 30) || !a || !b) return 0;
    return fp8_matmul_workspace_bytes((int)m, (int)n, (int)k, operand_of(a), operand_of(b));
}

int lb_fp8_matmul(lb_context *h, int64_t m, int64_t n, int64_t k, const lb_fp8_operand *a, const lb_fp8_operand *b, void *out, int dtype,
                  int64_t out_stride, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    REQUIRE(value_size(dtype), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
    REQUIRE(m >= 0 && n >= 0 && k >= 0 && m <= (1 << 30) && n <= (1 << 30) && k <= (1 << 30), "m, n or k is out of range");
    if ((rc = operand_ok(a, m, k)) || (rc = operand_ok(b, n, k))) return rc;
    if (m == 0 || n == 0) return LB_OK;
    REQUIRE(blocks_of(m) * ((n + 63) / 64) < (int64_t)1 << 31, "too many tiles for one call");
    if ((rc = rows_ok(out, m, n, out_stride, value_size(dtype)))) return rc;
    if (k == 0) { // an empty sum
        LB_CUDA(cudaMemset2DAsync(out, (size_t)(m > 1 ? out_stride : n) * value_size(dtype), 0, (size_t)n * value_size(dtype), (size_t)m, S(stream)));
        return LB_OK;
    }
    if ((rc = workspace_ok(workspace, workspace_bytes, lb_fp8_matmul_workspace_bytes(m, n, k, a, b)))) return rc;
    return fp8_matmul(C(h), (int)m, (int)n, (int)k, operand_of(a), operand_of(b), out, dtype, out_stride, workspace, S(stream));
}

// The tensors of a call that hold values, and for a client that has none one of no values
static std::vector<ClipPart> clip_parts(int n_clients, int n_tensors, const int *clients, const int *dtypes, const int64_t *sizes, const int *out_dtypes)
{
    std::vector<ClipPart> parts;
    parts.reserve((size_t)n_tensors + n_clients);
    auto type = [&](const int *types, int i) { return types && n_tensors ? types[i] : 1; };
    int i = 0;
    for (int k = 0; k < n_clients; ++k) {
        const size_t begin = parts.size();
        for (; i < n_tensors && clients[i] == k; ++i)
            if (sizes[i]) parts.push_back({nullptr, nullptr, (long)sizes[i], k, type(dtypes, i), type(out_dtypes, i), i});
        if (parts.size() == begin) parts.push_back({nullptr, nullptr, 0, k, type(dtypes, 0), type(out_dtypes, 0), -1});
    }
    return parts;
}

static int clip_ok(int n_clients, int n_tensors, const int *clients, const int *dtypes, const int64_t *sizes, const int *out_dtypes)
{
    REQUIRE(n_clients >= 0 && n_clients < 1 << 23 && n_tensors >= 0, "n_clients or n_tensors is out of range");
    REQUIRE(n_tensors == 0 || (clients && dtypes && sizes), "operand is null");
    double all = 0.0;
    for (int i = 0; i < n_tensors; ++i) {
        REQUIRE(clients[i] >= (i ? clients[i - 1] : 0) && clients[i] < n_clients, "the tensors are in the order of their clients");
        REQUIRE(sizes[i] >= 0 && sizes[i] <= (int64_t)1 << 40, "a tensor's size is out of range");
        REQUIRE(value_size(dtypes[i]) && (!out_dtypes || value_size(out_dtypes[i])), "dtype is 1 (float), 3 (bfloat16) or 4 (half)");
        all += (double)sizes[i];
    }
    REQUIRE(all <= (double)((int64_t)1 << 40), "too many values for one call");
    return LB_OK;
}

// No result may lie on another one, or on what is still to be read: in place, a tensor's result is the tensor itself
static int clip_apart(const std::vector<ClipPart> &parts)
{
    struct Span {
        uintptr_t begin, end;
        bool out;
    };
    std::vector<Span> spans;
    spans.reserve(2 * parts.size());
    uintptr_t low = UINTPTR_MAX, high = 0, last = 0;
    bool in_order = true;
    for (const ClipPart &p : parts)
        if (p.out) {
            const uintptr_t b = (uintptr_t)p.out, e = b + (uintptr_t)p.n * (uintptr_t)value_size(p.out_type);
            in_order = in_order && b >= last;
            last = e;
            low = b < low ? b : low;
            high = e > high ? e : high;
            spans.push_back({b, e, true});
        }
    if (spans.empty()) return LB_OK;
    bool clear = in_order;
    for (const ClipPart &p : parts)
        if (p.n && p.in != p.out) {
            const uintptr_t b = (uintptr_t)p.in, e = b + (uintptr_t)p.n * (uintptr_t)value_size(p.in_type);
            clear = clear && (e <= low || b >= high);
            spans.push_back({b, e, false});
        }
    if (clear) return LB_OK;
    std::sort(spans.begin(), spans.end(), [](const Span &x, const Span &y) { return x.begin < y.begin; });
    uintptr_t any = 0, out = 0;
    for (const Span &s : spans) {
        REQUIRE(s.begin >= (s.out ? any : out), "a result overlaps another one, or a tensor that is not its own");
        any = s.end > any ? s.end : any;
        if (s.out) out = s.end > out ? s.end : out;
    }
    return LB_OK;
}

static size_t clip_bytes(int n_clients, int n_tensors, const int64_t *sizes)
{
    size_t sums = (size_t)n_clients; // clients without values
    for (int i = 0; i < n_tensors; ++i) sums += sizes[i] ? clip_sums(sizes[i]) : 0;
    return sums * 8;
}

size_t lb_clip_updates_workspace_bytes(int n_clients, int n_tensors, const int64_t *sizes)
{
    if (n_clients < 1 || n_tensors < 0 || (n_tensors && !sizes)) return 0;
    for (int i = 0; i < n_tensors; ++i)
        if (sizes[i] < 0) return 0;
    return clip_bytes(n_clients, n_tensors, sizes);
}

int lb_clip_updates(lb_context *h, int n_clients, int n_tensors, const int *clients, const void *const *tensors, const int *dtypes,
                    const int64_t *sizes, double max_norm, void *const *outs, const int *out_dtypes, double *norms, void *workspace,
                    size_t workspace_bytes, void *stream)
try {
    int rc = bind(h);
    if (rc) return rc;
    if (!outs) out_dtypes = nullptr;
    if ((rc = clip_ok(n_clients, n_tensors, clients, dtypes, sizes, out_dtypes))) return rc;
    REQUIRE(max_norm >= 0.0, "max_norm is a number that is not negative");
    if (n_clients == 0) return LB_OK;
    REQUIRE(norms && (n_tensors == 0 || (tensors && (!outs || out_dtypes))), "operand is null");
    REQUIRE((uintptr_t)norms % 8 == 0, "an operand is not aligned to its type");
    std::vector<ClipPart> parts = clip_parts(n_clients, n_tensors, clients, dtypes, sizes, out_dtypes);
    for (ClipPart &p : parts) {
        const int i = p.index;
        if (i < 0) continue;
        REQUIRE(tensors[i] && (uintptr_t)tensors[i] % value_size(p.in_type) == 0, "a tensor is null or not aligned to its type");
        p.in = tensors[i];
        if (!outs) continue;
        REQUIRE(outs[i] && (uintptr_t)outs[i] % value_size(p.out_type) == 0, "a result is null or not aligned to its type");
        REQUIRE(outs[i] != tensors[i] || p.in_type == p.out_type, "a result in place has the type of its tensor");
        p.out = outs[i];
    }
    if ((rc = clip_apart(parts))) return rc;
    if ((rc = workspace_ok(workspace, workspace_bytes, clip_bytes(n_clients, n_tensors, sizes)))) return rc;
    return clip_updates(C(h), parts.data(), (int)parts.size(), outs != nullptr, max_norm, reinterpret_cast<double *>(workspace), norms, S(stream));
} catch (const std::bad_alloc &) {
    set_error("out of host memory");
    return LB_ERR_NO_MEMORY;
}

int lb_check_status(lb_context *h, void *stream)
{
    int rc = bind(h);
    if (rc) return rc;
    int flags = 0;
    LB_CUDA(cudaMemcpyAsync(&flags, C(h)->d_status, sizeof(int), cudaMemcpyDeviceToHost, S(stream)));
    LB_CUDA(cudaStreamSynchronize(S(stream)));
    if (flags) {
        LB_CUDA(cudaMemsetAsync(C(h)->d_status, 0, sizeof(int), S(stream)));
        std::string message;
        rc = status_of(flags, message);
        set_error(message);
    }
    return rc;
}

} // extern "C"
