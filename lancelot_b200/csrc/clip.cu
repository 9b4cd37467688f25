// The norms of clients' updates, each over many tensors, and the updates scaled down to a largest norm:
//
//   norm = sqrt(sum of v^2 over all tensors of a client)     f = min(1, most / norm), rounded to 32 bits; NaN where the norm is not finite     out = v * f
//
// A bound on the norm is the plain defence against an update that outweighs the others, next to the selection by distances
// (lancelot-main-GPU/utils/byzantine_fl.py:162-171,527-536); the reference has none.
//
// Squares of 32-bit floats are exact in 64 bits, and so are summed there: no sum passes the range, and small entries are not lost behind
// large ones.  The tensors are cut into pieces, a block each; a piece's sum goes to its own place, and every block that needs a client's norm adds
// its pieces' sums up in the same order, so that results do not depend on which block was first.
//
// The values of some clients (a round) are read for their sums by one kernel, and read again, the last ones first, and written by the next one, whose other
// blocks sum up the round after that.  Every kernel starts while its predecessor ends (programmatic launches).  Bound by memory: the norms of
// 20 x 11 M take 130 us (6.9 TB/s).  As flat rows 20 x 11 M take 403 us (floor 277): a third of the second reading misses L2 (61 MB of DRAM read for a
// client's 45), and a round's kernel has a start and an end of some microseconds.  Without rounds, every value read twice from DRAM, it takes 451 us,
// with rounds of one client 422, with sums and results in kernels of their own 425; a persistent kernel whose blocks meet between a round's two parts takes
// 480 us, 6 of them for each meeting.  In place 20 x 11 M take 389 us.  11 M values in bf16 as a row of 32 bits: 18.5 us; four clients of eight tensors: 4.3 us.
// Rounds are for tensors of one type: where types differ every run of like tensors is a launch, the sums of all clients first (20 x 11 M of 62 tensors that
// alternate between 16 and 32 bits: 7.3 ms).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "product.cuh"

namespace lb {

namespace {

constexpr int kThreads = 256;
constexpr int kMostTensors = 640;    // of one launch: they travel as its argument
constexpr int kLeastPiece = 1024;    // elements: clip_sums counts on it
constexpr double kRoundBytes = 96e6; // of values, unless a single client has more: most of them stay in L2 until they are read again

struct Part {
    const void *in;
    void *out; // NULL: nothing is written
    long n;
    int first;            // of the launch's pieces
    int slot;             // of that piece's sum
    int slots, slots_end; // of all sums of the client
    int client, begins;   // begins: whether it is the client's first tensor
};
template <int MOST> struct ClipArgs {
    Part tensor[MOST];
    int n_scale, n_tensors;       // the first n_scale tensors are written, the others are summed up
    int scale_piece, sum_piece;   // elements of their pieces
    int scale_pieces, sum_pieces; // how many
    double most;
    double *partial, *norms;
};

static_assert(sizeof(ClipArgs<kMostTensors>) <= 31 * 1024, "arguments and what the driver puts before them share 32 KB");

template <typename T> struct Pack; // values in 16 bytes
template <> struct Pack<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
    static __device__ __forceinline__ float one(float v) { return v; }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(x[i] << 16), v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ float one(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct Pack<__half> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float *v)
    {
        const unsigned x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float one(__half v) { return __half2float(v); }
};

// the sum of a block's values, in every thread; the order is fixed
__device__ __forceinline__ double block_sum(double v, double *shared)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) v += shared[i];
    return v;
}

// the tensor that holds a piece, of tensors lo to hi - 1
template <int MOST> __device__ __forceinline__ const Part &tensor_of(const ClipArgs<MOST> &a, int lo, int hi, int piece)
{
    --hi;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.tensor[mid].first <= piece) lo = mid;
        else hi = mid - 1;
    }
    return a.tensor[lo];
}

// The sum of squares of values from 16 bytes.  16-bit types: conversions to 64 bits come slowly (16 a cycle), so a value that is part of 20 bits is
// moved to its place in a double's upper half by hand; that is not right for zeros and for what is below 2^-126 (they come out as 2^-126 at
// most), which does not matter beside a value from 2^-60 on, nor for what is not finite.
__device__ __forceinline__ double add_squares(double sum, const float (&v)[4])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fma((double)v[e], (double)v[e], sum);
    return sum;
}
__device__ __forceinline__ double add_squares(double sum, const float (&v)[8])
{
    unsigned u[8], most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        u[e] = __float_as_uint(v[e]) & 0x7fffffffu;
        most = max(most, u[e]);
    }
    if (most - 0x21800000u < 0x7f800000u - 0x21800000u) { // 2^-60 and infinity
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double d = __hiloint2double((int)((u[e] >> 3) + 0x38000000u), 0);
            sum = fma(d, d, sum);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fma((double)v[e], (double)v[e], sum);
    }
    return sum;
}

template <typename T> __device__ __forceinline__ double squares(const T *p, int n)
{
    constexpr int N = Pack<T>::kN;
    double sum = 0.0;
    const int head = min((int)((16 - (unsigned)(uintptr_t)p % 16) % 16 / sizeof(T)), n), body = (n - head) / N * N;
    const T *q = p + head;
    for (int i = threadIdx.x * N; i < body; i += 4 * kThreads * N) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = i + j * kThreads * N < body ? __ldg(reinterpret_cast<const uint4 *>(q + i + j * kThreads * N)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[N];
            Pack<T>::open(w[j], v);
            sum = add_squares(sum, v);
        }
    }
    for (int i = threadIdx.x; i < n - body; i += kThreads) { // what lies before the first boundary and behind the last one
        const double v = Pack<T>::one(p[i < head ? i : i + body]);
        sum = fma(v, v, sum);
    }
    return sum;
}
// N values from `off` elements on behind a boundary of kAlign elements, out of the aligned pieces that they lie in: the pieces, and the values
template <typename T, int N> struct Raw { // 16-bit types
    static constexpr int kAlign = N, kSteps = N == 8 ? 3 : 4; // kSteps: of a thread, whose loads are on their way together
    unsigned w[N];
    __device__ __forceinline__ void part(const T *q, int at)
    {
        if constexpr (N == 8) {
            const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(q));
            w[at] = x.x, w[at + 1] = x.y, w[at + 2] = x.z, w[at + 3] = x.w;
        } else {
            const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(q));
            w[at] = x.x, w[at + 1] = x.y;
        }
    }
    __device__ __forceinline__ void load(const T *q, int off)
    {
        part(q, 0);
        if (off) part(q + N, N / 2);
    }
    __device__ __forceinline__ void open(int off, float (&v)[N])
    {
        if (off) {
            if constexpr (N == 8) {
#pragma unroll
                for (int e = 0; e < 6; ++e) w[e] = off & 4 ? w[e + 2] : w[e];
            }
#pragma unroll
            for (int e = 0; e <= N / 2; ++e)
                if (e + 1 < N) w[e] = off & 2 ? w[e + 1] : w[e];
#pragma unroll
            for (int e = 0; e < N / 2; ++e) w[e] = __funnelshift_r(w[e], w[e + 1], off & 1 ? 16 : 0);
        }
        float u[8];
        Pack<T>::open(make_uint4(w[0], w[1], N == 8 ? w[N - 6] : 0, N == 8 ? w[N - 5] : 0), u);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = u[e];
    }
};
template <int N> struct Raw<float, N> {
    static constexpr int kAlign = 4, kSteps = N == 4 ? 4 : 2;
    uint4 r[N / 4 + 1];
    __device__ __forceinline__ void load(const float *q, int off)
    {
#pragma unroll
        for (int j = 0; j < N / 4; ++j) r[j] = __ldcs(reinterpret_cast<const uint4 *>(q) + j);
        if (off) r[N / 4] = __ldcs(reinterpret_cast<const uint4 *>(q) + N / 4);
    }
    __device__ __forceinline__ void open(int off, float (&v)[N])
    {
        float w[N + 4];
#pragma unroll
        for (int j = 0; j <= N / 4; ++j) Pack<float>::open(r[j], w + 4 * j);
        if (off) {
#pragma unroll
            for (int e = 0; e < N + 2; ++e) w[e] = off & 2 ? w[e + 2] : w[e];
#pragma unroll
            for (int e = 0; e < N; ++e) w[e] = off & 1 ? w[e + 1] : w[e];
        }
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = w[e];
    }
};
__device__ __forceinline__ void store(float *p, const float (&v)[4]) { __stcs(reinterpret_cast<float4 *>(p), make_float4(v[0], v[1], v[2], v[3])); }
template <typename O> __device__ __forceinline__ void store(O *p, const float (&v)[8])
{
    __stcs(reinterpret_cast<uint4 *>(p), make_uint4(pack2(p, v[0], v[1]), pack2(p, v[2], v[3]), pack2(p, v[4], v[5]), pack2(p, v[6], v[7])));
}

// out = p * f, 16 bytes of results a thread and step.  A tensor seldom starts at the same place between two 16-byte boundaries as its run of the
// flat row: the results of a step are put together from the two or three aligned pieces that their values lie in.
template <typename T, typename O> struct Scaling {
    using R = Raw<T, 16 / sizeof(O)>;
    static constexpr int N = 16 / sizeof(O), A = R::kAlign, kStep = kThreads * N, kBatch = R::kSteps * kStep;
    const T *p;
    O *out;
    int n, off, first, from, body;
    R r[R::kSteps];

    __device__ __forceinline__ Scaling(const T *p_, O *out_, int n_) : p(p_), out(out_), n(n_)
    {
        const int head = min((int)((16 - (unsigned)(uintptr_t)out % 16) % 16 / sizeof(O)), n);
        off = (int)((unsigned)((uintptr_t)(p + head) / sizeof(T)) % A); // of the values of the first step
        first = off <= head ? head : head + N;                          // pieces that begin before p are not read
        int steps = max((n - first) / N, 0);
        if (off && steps > 0 && first + N * steps - off + A > n) --steps; // nor those that end behind its end
        body = steps * N;
        from = min(first, n);
    }
    __device__ __forceinline__ void load(int i) // all loads of a batch before its first store: none may pass one that might lie in its way
    {
#pragma unroll
        for (int j = 0; j < R::kSteps; ++j)
            if (i + j * kStep < body) r[j].load(p + first - off + i + j * kStep, off);
    }
    __device__ __forceinline__ void finish(int i, float f) // with the batch from i on loaded
    {
        while (true) {
#pragma unroll
            for (int j = 0; j < R::kSteps; ++j)
                if (i + j * kStep < body) {
                    float v[N];
                    r[j].open(off, v);
#pragma unroll
                    for (int e = 0; e < N; ++e) v[e] *= f;
                    store(out + first + i + j * kStep, v);
                }
            i += kBatch;
            if (i >= body) break;
            load(i);
        }
        for (int k = threadIdx.x; k < n - body; k += kThreads) {
            const int j = k < from ? k : k + body;
            put(out + j, Pack<T>::one(p[j]) * f);
        }
    }
};

// what the kernel before this one wrote is there
__device__ __forceinline__ void predecessor_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// the next kernel's blocks may come as soon as there is room
__device__ __forceinline__ void successor_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T, int MOST> __device__ __forceinline__ void sum_up(const ClipArgs<MOST> &a, int i, double *shared)
{
    const Part &t = tensor_of(a, a.n_scale, a.n_tensors, i);
    const long e = (long)(i - t.first) * a.sum_piece;
    const double sum = block_sum(squares(reinterpret_cast<const T *>(t.in) + e, (int)min((long)a.sum_piece, t.n - e)), shared);
    if (threadIdx.x == 0) a.partial[t.slot + (i - t.first)] = sum;
    predecessor_done(); // nothing of it is used: whoever waits for this kernel has then waited for that one too
}
template <typename T, int MOST> __global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ ClipArgs<MOST> a)
{
    __shared__ double shared[kThreads / 32];
    successor_may_start();
    sum_up<T>(a, (int)blockIdx.x, shared);
}

__device__ __forceinline__ double norm_of(const double *partial, int from, int to, double *shared)
{
    double sum = 0.0;
    for (int j = from + (int)threadIdx.x; j < to; j += kThreads) sum += __ldcg(partial + j);
    return sqrt(block_sum(sum, shared));
}

// Blocks that write the results of some clients, and blocks that sum up the next clients' values, by turns: memory is read and written at once
template <typename T, typename O, int MOST> __global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ ClipArgs<MOST> a)
{
    __shared__ double shared[kThreads / 32];
    successor_may_start();
    const int pairs = min(a.scale_pieces, a.sum_pieces), block = (int)blockIdx.x;
    const bool sums = block < 2 * pairs ? block & 1 : a.sum_pieces > pairs;
    int i = block < 2 * pairs ? block >> 1 : block - pairs;
    if (sums) {
        sum_up<T>(a, i, shared);
        return;
    }
    i = a.scale_pieces - 1 - i; // what was read last is read first
    const Part &t = tensor_of(a, 0, a.n_scale, i);
    const long e = (long)(i - t.first) * a.scale_piece;
    // values on their way while the norm is found: no kernel before this one that may still run writes them
    Scaling<T, O> s(reinterpret_cast<const T *>(t.in) + e, t.out ? reinterpret_cast<O *>(t.out) + e : nullptr, (int)min((long)a.scale_piece, t.n - e));
    s.load(threadIdx.x * s.N);
    predecessor_done();
    const double norm = norm_of(a.partial, t.slots, t.slots_end, shared);
    if (threadIdx.x == 0 && t.begins && i == t.first) a.norms[t.client] = norm;
    const float f = !isfinite(norm) ? __int_as_float(0x7fc00000) : norm > a.most ? (float)(a.most / norm) : 1.0f;
    if (!t.out || (f == 1.0f && t.out == t.in)) return;
    s.finish(threadIdx.x * s.N, f);
}

// norms alone: a block for a client
struct Client {
    int client, slots, slots_end;
};
constexpr int kMostClients = 2000;
struct NormArgs {
    Client client[kMostClients];
    const double *partial;
    double *norms;
};
__global__ void __launch_bounds__(kThreads) norms_kernel(const __grid_constant__ NormArgs a)
{
    __shared__ double shared[kThreads / 32];
    const Client c = a.client[blockIdx.x];
    predecessor_done();
    const double norm = norm_of(a.partial, c.slots, c.slots_end, shared);
    if (threadIdx.x == 0) a.norms[c.client] = norm;
}

// A launch: tensors of the same types; whole clients where a client's tensors fit and are of the same types
struct Launch {
    int first, count; // of the tensors
    int piece, pieces;
    bool writes; // a launch of sums, or of results
};

double part_bytes(const ClipPart &p) { return (double)p.n * (p.in_type == 1 ? 4 : 2); }

// The launches of a call, and their tables
void plan(const Context *ctx, const ClipPart *in, int n, bool writes, std::vector<Launch> &launches, std::vector<Part> &parts)
{
    long slots = 0;
    auto pieces_of = [](long size, int piece) { return size ? (int)((size + piece - 1) / piece) : 1; };
    auto add = [&](int i, int end) { // the sums of some tensors
        double all = 0.0;
        for (int j = i; j < end; ++j) all += (double)in[j].n;
        // some eight pieces an SM, of 64 KB of 32-bit values at most: every block of the second kernel reads the sums of all pieces of its client
        const double even = all / (8.0 * ctx->sm_count);
        const int piece = even <= kLeastPiece ? kLeastPiece : even >= 16384 && all < 16384.0 * (1 << 20) ? 16384 : ((int)(even / 1024) + 1) * 1024;
        Launch l = {i, end - i, piece, 0, false};
        for (int j = i; j < end; ++j) {
            const int pieces = pieces_of(in[j].n, piece);
            parts[j] = {in[j].in, in[j].out, in[j].n, l.pieces, (int)slots, 0, (int)slots + pieces, in[j].client, j == 0 || in[j].client != in[j - 1].client};
            l.pieces += pieces;
            slots += pieces;
        }
        launches.push_back(l);
    };
    auto alike = [&](int i, int j) { return in[i].in_type == in[j].in_type && in[i].out_type == in[j].out_type; };
    bool same = true;
    for (int i = 1; i < n; ++i) same = same && alike(i - 1, i);
    for (int i = 0; i < n;) {
        // as many whole clients as one launch holds and L2 keeps; where there is none, because a client has more tensors or types differ, all tensors
        int whole = i;
        double bytes = 0.0;
        for (int end = i; same && end < n && end - i < kMostTensors; ++end) {
            bytes += part_bytes(in[end]);
            if (end + 1 < n && in[end + 1].client == in[end].client) continue;
            if (writes && whole > i && bytes > kRoundBytes) break;
            whole = end + 1;
        }
        const size_t first = launches.size();
        if (whole > i) {
            add(i, whole);
        } else {
            whole = n;
            for (int j = i, end; j < n; j = end) {
                for (end = j; end < n && end - j < kMostTensors && alike(end, j);) ++end;
                add(j, end);
            }
        }
        if (writes)
            for (size_t j = first, last = launches.size(); j < last; ++j) {
                const Launch sums = launches[j];
                launches.push_back(sums);
                launches.back().writes = true;
            }
        i = whole;
    }
    for (int i = 0; i < n;) { // a client's sums lie together, those of several launches too
        int end = i;
        while (end < n && in[end].client == in[i].client) ++end;
        for (int j = i; j < end; ++j) parts[j].slots = parts[i].slot, parts[j].slots_end = parts[end - 1].slots_end;
        i = end;
    }
}

// The first kernel of a call waits for what came before it; the others are set up, and those of sums begin, while their predecessor ends
int start(const void *kernel, int grid, void *args, bool first, cudaStream_t stream)
{
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)grid);
    c.blockDim = dim3(kThreads);
    c.stream = stream;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &early;
    c.numAttrs = first ? 0 : 1;
    void *list[] = {args};
    LB_CUDA(cudaLaunchKernelExC(&c, kernel, list));
    return LB_OK;
}
template <int MOST>
int launch(const std::vector<Part> &parts, const Launch &l, const Launch *next, const void *kernel, double most, double *partial, double *norms, bool first, cudaStream_t stream)
{
    ClipArgs<MOST> a;
    const int count = l.count + (next ? next->count : 0);
    std::copy(parts.begin() + l.first, parts.begin() + l.first + count, a.tensor);
    const Launch *sums = l.writes ? next : &l;
    a.n_scale = l.writes ? l.count : 0;
    a.n_tensors = count;
    a.scale_piece = l.piece;
    a.scale_pieces = l.writes ? l.pieces : 0;
    a.sum_piece = sums ? sums->piece : 0;
    a.sum_pieces = sums ? sums->pieces : 0;
    a.most = most;
    a.partial = partial;
    a.norms = norms;
    return start(kernel, a.scale_pieces + a.sum_pieces, &a, first, stream);
}
template <typename T, int MOST> const void *kernel_of(int out_type)
{
    return out_type == 0   ? reinterpret_cast<const void *>(norm_kernel<T, MOST>)
           : out_type == 1 ? reinterpret_cast<const void *>(clip_kernel<T, float, MOST>)
           : out_type == 3 ? reinterpret_cast<const void *>(clip_kernel<T, __nv_bfloat16, MOST>)
                           : reinterpret_cast<const void *>(clip_kernel<T, __half, MOST>);
}
template <int MOST> const void *kernel_of(int in_type, int out_type)
{
    return in_type == 1 ? kernel_of<float, MOST>(out_type) : in_type == 3 ? kernel_of<__nv_bfloat16, MOST>(out_type) : kernel_of<__half, MOST>(out_type);
}

} // namespace

int clip_updates(const Context *ctx, const ClipPart *in, int n, bool writes, double most, double *partial, double *norms, cudaStream_t stream)
{
    std::vector<Launch> launches;
    launches.reserve(8);
    std::vector<Part> parts(n);
    plan(ctx, in, n, writes, launches, parts);
    int rc = LB_OK;
    for (size_t j = 0; j < launches.size(); ++j) {
        const Launch &l = launches[j];
        const bool first = j == 0;
        // the results of some clients go with the sums of the next ones
        const Launch *next = l.writes && j + 1 < launches.size() && !launches[j + 1].writes && l.count + launches[j + 1].count <= kMostTensors &&
                                     l.first + l.count == launches[j + 1].first && in[l.first].in_type == in[launches[j + 1].first].in_type
                                 ? &launches[++j]
                                 : nullptr;
        double bytes = 0.0;
        const int count = l.count + (next ? next->count : 0);
        for (int i = l.first; i < l.first + count; ++i)
            bytes += !l.writes || i >= l.first + l.count ? part_bytes(in[i]) : in[i].out ? (double)in[i].n * (in[i].out_type == 1 ? 4 : 2) : 0.0;
        count_launch(l.writes ? "clip_scale" : "clip_norm", stream, bytes);
        const int in_type = in[l.first].in_type, out_type = l.writes ? in[l.first].out_type : 0;
        if (count <= 32) rc = launch<32>(parts, l, next, kernel_of<32>(in_type, out_type), most, partial, norms, first, stream);
        else if (count <= 128) rc = launch<128>(parts, l, next, kernel_of<128>(in_type, out_type), most, partial, norms, first, stream);
        else rc = launch<kMostTensors>(parts, l, next, kernel_of<kMostTensors>(in_type, out_type), most, partial, norms, first, stream);
        if (rc) return rc;
    }
    if (writes) return LB_OK;
    NormArgs a;
    a.partial = partial;
    a.norms = norms;
    int held = 0;
    for (int i = 0; i < n; ++i) {
        if (parts[i].begins) a.client[held++] = {parts[i].client, parts[i].slots, parts[i].slots_end};
        if (held < kMostClients && (i + 1 < n || held == 0)) continue;
        count_launch("clip_norms", stream, 0.0);
        if ((rc = start(reinterpret_cast<const void *>(norms_kernel), held, &a, false, stream))) return rc;
        held = 0;
    }
    return LB_OK;
}

} // namespace lb
