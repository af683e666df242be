// host_operators.h -- C entry points of the stand-alone operators (gated_delta.h, w4_matvec.h): device pointers, the caller's stream, nothing
// allocated, nothing waited for, so that every call can be captured into a graph.  Arguments are checked before anything is launched.

namespace {
struct OpDevice {                                 // the call's device for as long as it runs, the caller's afterwards
    int before = -1; hipError_t err;
    explicit OpDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OpDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

struct OpSpan { const char* lo; const char* hi; };
OpSpan op_span(const void* p, const long* stride, const long* size, int dims, long last, int elem) {
    long n = last;
    for (int i = 0; i < dims; ++i) n += (size[i] - 1) * stride[i];
    return {(const char*)p, (const char*)p + n * elem};
}
bool op_meet(const OpSpan& x, const OpSpan& y) { return x.lo < y.hi && y.lo < x.hi; }
// no two elements of an output in one place: every dimension steps over all that the smaller steps span
bool op_apart(const long* stride, const long* size, int dims, long last) {
    bool used[3] = {false, false, false};
    long span = last;
    for (int k = 0; k < dims; ++k) {
        int best = -1;
        for (int i = 0; i < dims; ++i) if (!used[i] && (best < 0 || stride[i] < stride[best] || (stride[i] == stride[best] && size[i] < size[best]))) best = i;
        used[best] = true;
        if (size[best] == 1) continue;
        if (stride[best] < span) return false;
        span += (size[best] - 1) * stride[best];
    }
    return true;
}
constexpr long OP_THREADS = 0xffffffffL;          // of a launch, in one dimension
int op_bytes(int dtype) { return dtype == DPDF_F32 ? 4 : dtype == DPDF_F16 || dtype == DPDF_BF16 ? 2 : 0; }
bool op_aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

int gd_columns(int Dk, int Dv, int dtype) { return Dv <= 32 && Dk <= 64 && dtype == DPDF_F32 ? 32 : Dv <= 64 ? 64 : 128; }
int gd_columns(const GatedDeltaArgs& a, int dtype) { return gd_columns(a.Dk, a.Dv, dtype); }
int gd_check(const dpdf_gated_delta_args* p, bool step, GatedDeltaArgs& a) {
    if (!p) return set_err(DPDF_E_INVALID, "null argument");
    const dpdf_gated_delta_args& x = *p;
    const int e = op_bytes(x.dtype), ge = op_bytes(x.gate_dtype);
    if (!e || !ge || (x.gate_dtype != DPDF_F32 && x.gate_dtype != x.dtype)) return set_err(DPDF_E_INVALID, "gated delta rule: unsupported dtypes %d / %d", x.dtype, x.gate_dtype);
    if (x.batch < 0 || x.frames < 0) return set_err(DPDF_E_INVALID, "gated delta rule: negative size batch=%d frames=%d", x.batch, x.frames);
    if (x.frames > 1 << 30) return set_err(DPDF_E_INVALID, "gated delta rule: %d frames are too large a number for one call", x.frames);
    if (x.k_heads < 1 || x.v_heads < 1 || x.v_heads % x.k_heads) return set_err(DPDF_E_INVALID, "gated delta rule: %d value heads are no multiple of %d key heads", x.v_heads, x.k_heads);
    // kernels count columns, inputs and outputs with 32 bits and go some hundred behind the last
    if (x.k_dim < 1 || x.k_dim > 128 || x.v_dim < 1 || x.v_dim > 1 << 28) return set_err(DPDF_E_INVALID, "gated delta rule: head sizes %d (1 .. 128) and %d (1 .. 2^28)", x.k_dim, x.v_dim);
    if (!(x.scale - x.scale == 0.f)) return set_err(DPDF_E_INVALID, "gated delta rule: scale is not finite");
    if (step && x.lengths) return set_err(DPDF_E_INVALID, "gated delta rule: a step takes no lengths");
    if (!step && x.active) return set_err(DPDF_E_INVALID, "gated delta rule: clips take no mask of active streams");
    const long B = x.batch, T = x.frames, Hk = x.k_heads, Hv = x.v_heads, Dk = x.k_dim, Dv = x.v_dim;
    // one wave to 32 columns of a hop, columns / 16 waves to as many of a clip; B Hv is below 2^62
    const long columns = step ? 32 : gd_columns(x.k_dim, x.v_dim, x.dtype), threads = step ? 64 : 4 * columns;
    if (B * Hv > OP_THREADS / threads || (Dv + columns - 1) / columns > OP_THREADS / threads / (B * Hv > 0 ? B * Hv : 1)) return set_err(DPDF_E_INVALID, "gated delta rule: batch %d with %d heads of %d is too large for one call", x.batch, x.v_heads, x.v_dim);
    if (B && (step && (!x.state_in || !x.state_out))) return set_err(DPDF_E_INVALID, "gated delta rule: a step needs its state");
    const long kd[3] = {B, T, Hk}, vd[3] = {B, T, Hv};
    for (const long* s : {x.q_stride, x.k_stride, x.v_stride, x.g_stride, x.beta_stride, x.out_stride})
        for (int i = 0; i < 3; ++i) if (s[i] < 0) return set_err(DPDF_E_INVALID, "gated delta rule: negative stride");
    const long n = B * Hv * Dk * Dv * 4;
    const OpSpan si = {(const char*)x.state_in, (const char*)x.state_in + (x.state_in ? n : 0)}, so = {(const char*)x.state_out, (const char*)x.state_out + (x.state_out ? n : 0)};
    const OpSpan len = {(const char*)x.lengths, (const char*)x.lengths + (x.lengths ? B * 4 : 0)}, act = {(const char*)x.active, (const char*)x.active + (x.active ? B : 0)};
    if (B && T) {
        if (!x.q || !x.k || !x.v || !x.g || !x.beta || !x.out) return set_err(DPDF_E_INVALID, "null argument");
        if (!op_aligned(x.q, e) || !op_aligned(x.k, e) || !op_aligned(x.v, e) || !op_aligned(x.out, e) || !op_aligned(x.g, ge) || !op_aligned(x.beta, ge))
            return set_err(DPDF_E_INVALID, "gated delta rule: a pointer is not aligned to its type");
        if (!op_apart(x.out_stride, vd, 3, Dv)) return set_err(DPDF_E_INVALID, "gated delta rule: elements of out share memory");
        const OpSpan o = op_span(x.out, x.out_stride, vd, 3, Dv, e);
        const OpSpan in[5] = {op_span(x.q, x.q_stride, kd, 3, Dk, e), op_span(x.k, x.k_stride, kd, 3, Dk, e), op_span(x.v, x.v_stride, vd, 3, Dv, e),
                              op_span(x.g, x.g_stride, vd, 3, 1, ge), op_span(x.beta, x.beta_stride, vd, 3, 1, ge)};
        for (const OpSpan& i : in) if (op_meet(o, i) || op_meet(so, i)) return set_err(DPDF_E_INVALID, "gated delta rule: an output overlaps an input");
        if (op_meet(o, si) || op_meet(o, so)) return set_err(DPDF_E_INVALID, "gated delta rule: out overlaps a state");
        if (op_meet(o, len) || op_meet(o, act)) return set_err(DPDF_E_INVALID, "gated delta rule: an output overlaps an input");
    }
    if (op_meet(so, len) || op_meet(so, act)) return set_err(DPDF_E_INVALID, "gated delta rule: an output overlaps an input");
    if (x.state_in != x.state_out && op_meet(si, so)) return set_err(DPDF_E_INVALID, "gated delta rule: the states overlap in part");
    if (!op_aligned(x.state_in, 4) || !op_aligned(x.state_out, 4) || !op_aligned(x.lengths, 4)) return set_err(DPDF_E_INVALID, "gated delta rule: a pointer is not aligned to its type");
    a.q = x.q; a.k = x.k; a.v = x.v; a.g = x.g; a.beta = x.beta; a.out = x.out;
    a.state_in = x.state_in; a.state_out = x.state_out; a.lengths = x.lengths; a.active = x.active;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = x.q_stride[i]; a.ks[i] = x.k_stride[i]; a.vs[i] = x.v_stride[i];
        a.gs[i] = x.g_stride[i]; a.bs[i] = x.beta_stride[i]; a.os[i] = x.out_stride[i];
    }
    // one frame has no next one: its step may be anything, but the rows that a chunk has behind it must lie behind it
    if (x.frames == 1) { a.qs[1] = a.ks[1] = Dk; a.vs[1] = a.os[1] = Dv; }
    a.B = x.batch; a.T = x.frames; a.Hk = x.k_heads; a.Hv = x.v_heads; a.Dk = x.k_dim; a.Dv = x.v_dim; a.scale = x.scale; a.gate = x.gate_dtype;
    a.segments = 1; a.seg = 0; a.starts = a.moves = nullptr; a.whole = a.even = a.sorted = 0; a.strips = 0;
    return DPDF_OK;
}

template <typename T>
void gd_launch_step(const GatedDeltaArgs& a, unsigned grid, hipStream_t s) {
#define GD_STEP(D) (a.whole ? (gated_delta_step_kernel<T, D, true><<<grid, 64, 0, s>>>(a)) : (gated_delta_step_kernel<T, D, false><<<grid, 64, 0, s>>>(a)))
    if (a.Dk <= 16) GD_STEP(16); else if (a.Dk <= 32) GD_STEP(32); else if (a.Dk <= 64) GD_STEP(64); else if (a.Dk <= 96) GD_STEP(96); else GD_STEP(128);
#undef GD_STEP
}
// Rows that can be read and written in pieces: whole fours of bytes
bool gd_fours(const void* p, const long (&s)[3], int e) { return op_aligned(p, 4) && s[0] * e % 4 == 0 && s[1] * e % 4 == 0 && s[2] * e % 4 == 0; }
void gd_pieces(GatedDeltaArgs& a, int e) {
    a.whole = a.Dk % 8 == 0 && gd_fours(a.q, a.qs, e) && gd_fours(a.k, a.ks, e);
    a.even = a.Dv % 4 == 0 && gd_fours(a.out, a.os, e);
}
// The frames of a chunk, the columns of a workgroup (gd_columns) and the workgroups that a CU holds at once (registers and LDS).  Two waves for 32 columns
// where a chunk has two diagonal blocks for them: with four, half of them would have no column (104 clips of 821 to 2463 frames, 8 heads of 16, fp32:
// 427 us with four, 343 with two; 30 of 700 frames, 8 heads of 48 x 32: 112 and 103; fp16 with its four blocks, 166 clips x 450 frames: 107 with four, 120 with two).
int gd_chunk(int dtype) { return dtype == DPDF_F32 ? 32 : 64; }
int gd_resident(const GatedDeltaArgs& a, int dtype) {
    const int columns = gd_columns(a, dtype);
    return columns == 128 || (a.Dk > 64 && dtype == DPDF_F16) ? 1 : columns == 64 ? 2 : a.Dk <= 32 ? 4 : 3;
}
// Segments for `heads` heads: as many as fill the chip once, and only where the chip would hold three times the workgroups there are.  A segment costs
// its frames about one and a half times more and a step of the join, a seventh of a chunk: hence no more than the root of five times the
// chunks (6 heads, 50 chunks: 67 us in 10 segments, 60 in 13, 56 in 17, 60 in 25; 3 heads, 100 chunks: 81 in 17, 76 in 20, 83 in 50), and at least two
// chunks each, four where the second pass would start in several rounds (2 clips of 17 chunks, 4 heads: 43 us by three, 59 by five;
// 111 heads, 14 chunks: 94 by two, 75 by five, 80 in one piece).
int gd_segments(const GatedDeltaArgs& a, int dtype, long heads, int cus) {
    const long strips = (a.Dv + gd_columns(a, dtype) - 1) / gd_columns(a, dtype), groups = heads * strips, room = (long)cus * gd_resident(a, dtype);
    const long chunks = ((long)a.T + gd_chunk(dtype) - 1) / gd_chunk(dtype);
    long n = room / groups;
    if (n > chunks / (groups * 4 > cus ? 4 : 2)) n = chunks / (groups * 4 > cus ? 4 : 2);
    while (n > 1 && n * n > 5 * chunks) --n;
    return n < 3 ? 1 : (int)n;
}
size_t gd_workspace(const GatedDeltaArgs& a, long heads, int segments) {
    return segments < 2 ? 0 : (size_t)segments * heads * a.Dk * (a.Dk + a.Dv) * sizeof(float);
}
template <typename T, int DKP, int NW>
void gd_launch_clip(GatedDeltaArgs& a, long heads, hipStream_t s) {
    constexpr int C = sizeof(T) == 4 ? 32 : 64;
    const long units = heads * a.segments, vcols = (a.Dv + 15) & ~15, kcols = (a.Dk + 15) & ~15;
    if (a.segments > 1) {
        a.strips = (int)((vcols + kcols + 16 * NW - 1) / (16 * NW));
        gated_delta_clip_kernel<T, DKP, NW, C, true><<<(unsigned)(units * a.strips), 64 * NW, 0, s>>>(a);
        a.strips = (int)(vcols / 16);
        gated_delta_join_kernel<DKP><<<(unsigned)(heads * a.strips), 4 * DKP, 0, s>>>(a, heads);
    }
    a.strips = (a.Dv + 16 * NW - 1) / (16 * NW);
    gated_delta_clip_kernel<T, DKP, NW, C, false><<<(unsigned)(units * a.strips), 64 * NW, 0, s>>>(a);
}
template <typename T>
void gd_launch_clips(GatedDeltaArgs& a, long heads, hipStream_t s) {
    constexpr bool F32 = sizeof(T) == 4;
    const int columns = gd_columns(a, F32 ? DPDF_F32 : DPDF_F16);
#define GD_CLIP(D) (columns == 64 ? gd_launch_clip<T, D, 4>(a, heads, s) : gd_launch_clip<T, D, 8>(a, heads, s))
    if constexpr (F32)
        if (columns == 32) return a.Dk <= 32 ? gd_launch_clip<T, 32, 2>(a, heads, s) : gd_launch_clip<T, 64, 2>(a, heads, s);
    if (a.Dk <= 32) GD_CLIP(32); else if (a.Dk <= 64) GD_CLIP(64); else GD_CLIP(128);
#undef GD_CLIP
}
template <typename F> void gd_type(int dtype, F f) {
    if (dtype == DPDF_F32) f(float()); else if (dtype == DPDF_F16) f(__half()); else f(__hip_bfloat16());
}
// calls f with the types of the values and of the gates
template <typename F> void gd_types(int dtype, int gate, F f) {
    if (dtype == DPDF_F32) f(float(), float());
    else if (dtype == DPDF_F16) { if (gate == DPDF_F32) f(__half(), float()); else f(__half(), __half()); }
    else { if (gate == DPDF_F32) f(__hip_bfloat16(), float()); else f(__hip_bfloat16(), __hip_bfloat16()); }
}

// Tiles of 16 outputs to a workgroup (nt) and its waves (nw), by the tiles that there are for each CU: few where the chip would not be full, many
// so that x is read less often.  us with nt of 1, 2, 4, weights from HBM, K = 4096 and 128 to a group where nothing else is said:
//     up to one for each CU    1.0: 8 rows of bf16 6.5, 8.2, 12.3; 2 of fp32 8.6, 10.7, 16.8; 8 of fp16, group 32 7.2, 10.3, 16.1
//     up to two                1.2: 1 of bf16, K = 8192 13.8, 12.8, 20.4; 1.8: 4 of fp16, group 64 10.5, 9.2, 14.2; 2.0: 2 of fp32 13.8, 12.0, 18.2
//     more                     3.5: 8 of bf16 18.2, 14.6, 14.0; 6: 2 of fp32 35.5, 31.8, 29.0; 8: 16 of bf16, K = 1024, group 64 26.7, 22.4, 10.7
// The last round of workgroups counts whole: with long sums of 16-bit rows, which are bound by reading codes, two are better where four would leave
// more of it empty (5: 8 of bf16 22.2, 19.6, 22.8; 10: 1 of bf16, K = 8192 56.6, 48.2, 53.5; but 1 of bf16, K = 1024 18.4, 14.2, 10.8; 16: 8 of bf16 62.4, 47.1, 43.5),
// and for one row or two, whose x costs little, up to eight (4: 15.1, 12.5, 14.1; 8: 27.3, 22.3, 23.3; with 4 rows, K = 8192, 3: 23.1, 23.2, 22.0).
// With four tiles, four waves, of which two workgroups fit on a CU and start at once (6: 2 of fp32 29.0 us, with eight waves 32.0), but eight where fp32
// rows have one workgroup to a CU at most (3.5: 18.7, with eight 17.1; 8 of bf16 14.0 and 14.3).
struct W4Split { int nt, nw; };
W4Split w4_split(const W4Args& a, int dtype, int cus) {
    const long tiles = ((long)a.N + 15) / 16 * (((long)a.M + 15) / 16), units = ((long)a.K + 127) / 128;
    int nt = tiles <= cus ? 1 : tiles <= 2L * cus ? 2 : 4, nw = W4_WAVES;
    if (nt == 4 && dtype != DPDF_F32 && a.group % 128 == 0 && a.K >= 4096 && tiles <= 10L * cus) {
        const long two = (tiles + 2 * cus - 1) / (2 * cus) * 2, four = (tiles + 4 * cus - 1) / (4 * cus) * 4;
        if (two < four || (a.M <= 2 && tiles <= 8L * cus)) nt = 2;
    }
    if (nt == 4 && (dtype != DPDF_F32 || tiles > 4L * cus)) nw = W4_WAVES / 2;
    return {nt, (int)(units < nw ? units : nw)};
}
template <typename T, typename G>
void w4_launch(const W4Args& a, unsigned grid, W4Split split, hipStream_t s) {
    const int nt = split.nt, nw = split.nw;
#define W4_RUN_(R, N) w4_matvec_kernel<T, G, R, N><<<grid, 64 * nw, 0, s>>>(a)
#define W4_RUN(R) (nt == 4 ? (W4_RUN_(R, 4)) : nt == 2 ? (W4_RUN_(R, 2)) : (W4_RUN_(R, 1)))
    if (a.group % 128 == 0) W4_RUN(4); else if (a.group % 64 == 0) W4_RUN(2); else W4_RUN(1);
#undef W4_RUN
#undef W4_RUN_
}

int w4_check(int dtype, long K, long N, int group, const char* what) {
    if (!op_bytes(dtype)) return set_err(DPDF_E_INVALID, "%s: unsupported dtype %d", what, dtype);
    if (K < 1 || N < 1) return set_err(DPDF_E_INVALID, "%s: empty layer %ld x %ld", what, N, K);
    if (K > 1 << 30 || N > 1 << 30) return set_err(DPDF_E_INVALID, "%s: a layer of %ld x %ld is too large", what, N, K);
    if (group < 32 || group % 32) return set_err(DPDF_E_INVALID, "%s: group %d is no multiple of 32", what, group);
    return DPDF_OK;
}
}  // namespace

extern "C" size_t dpdf_gated_delta_workspace(int device, const dpdf_gated_delta_args* args) {
    GatedDeltaArgs a;
    int cus = 0;
    if (gd_check(args, false, a) || !args->batch || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) return 0;
    const long heads = (long)args->batch * a.Hv;
    return gd_workspace(a, heads, gd_segments(a, args->dtype, heads, cus));
}

extern "C" int dpdf_gated_delta(int device, const dpdf_gated_delta_args* args, void* workspace, size_t workspace_bytes, void* stream) {
    GatedDeltaArgs a;
    if (int rc = gd_check(args, false, a)) return rc;
    if (!args->batch || (!args->frames && !args->state_out)) return DPDF_OK;
    // a chunk's rows, also those behind the last frame, are addressed with 32 bits
    const long most = (1L << 31) - 1, e = op_bytes(args->dtype);
    for (const long* s : {a.qs, a.ks, a.vs, a.os})
        if (s[1] > (most - (long)(a.Dk > a.Dv ? a.Dk : a.Dv) * e) / (64 * e)) return set_err(DPDF_E_INVALID, "gated delta rule: a stride of %ld from frame to frame is too large", s[1]);
    if (!op_aligned(workspace, 16)) return set_err(DPDF_E_INVALID, "gated delta rule: the workspace is not aligned to 16 bytes");
    gd_pieces(a, (int)e);
    OpDevice dev(device);
    HIP_TRY(dev.err);
    const long heads = (long)args->batch * a.Hv, chunk = gd_chunk(args->dtype);
    a.segments = 1; a.seg = (int)((args->frames + chunk - 1) / chunk * chunk);
    if (workspace) {
        int cus = 0;
        HIP_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
        const int n = gd_segments(a, args->dtype, heads, cus);
        if (n > 1 && workspace_bytes >= gd_workspace(a, heads, n)) {
            const long chunks = (args->frames + chunk - 1) / chunk, each = (chunks + n - 1) / n;
            a.seg = (int)(each * chunk); a.segments = (int)((chunks + each - 1) / each);
            const OpSpan ws = {(const char*)workspace, (const char*)workspace + gd_workspace(a, heads, a.segments)};
            const long B = args->batch, T = args->frames, kd[3] = {B, T, a.Hk}, vd[3] = {B, T, a.Hv}, ge = op_bytes(args->gate_dtype), state = heads * a.Dk * a.Dv * 4;
            const OpSpan other[9] = {op_span(a.q, a.qs, kd, 3, a.Dk, e), op_span(a.k, a.ks, kd, 3, a.Dk, e), op_span(a.v, a.vs, vd, 3, a.Dv, e), op_span(a.out, a.os, vd, 3, a.Dv, e),
                                     op_span(a.g, a.gs, vd, 3, 1, ge), op_span(a.beta, a.bs, vd, 3, 1, ge),
                                     {(const char*)a.state_in, (const char*)a.state_in + (a.state_in ? state : 0)}, {(const char*)a.state_out, (const char*)a.state_out + (a.state_out ? state : 0)},
                                     {(const char*)a.lengths, (const char*)a.lengths + (a.lengths ? B * 4 : 0)}};
            for (const OpSpan& o : other) if (op_meet(ws, o)) return set_err(DPDF_E_INVALID, "gated delta rule: the workspace overlaps a tensor");
            a.starts = (float*)workspace; a.moves = a.starts + (size_t)a.segments * heads * a.Dk * a.Dv;
        }
    }
    if (a.lengths && a.segments == 1 && a.B <= 4 * gd_columns(a, args->dtype) && a.B <= GD_RANKED && a.T < 1 << 25) {
        int cus = 0;
        HIP_TRY(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
        // all of them start at once otherwise (256 clips of 334 to 1003 frames, 4 heads of 64 in bf16: 210 us in the batch's order, 175 us so); of more clips than threads, the batch's order stays
        a.sorted = heads * ((a.Dv + gd_columns(a, args->dtype) - 1) / gd_columns(a, args->dtype)) > (long)cus * gd_resident(a, args->dtype);
    }
    gd_type(args->dtype, [&](auto t) { gd_launch_clips<decltype(t)>(a, heads, (hipStream_t)stream); });
    HIP_TRY(hipGetLastError());
    return DPDF_OK;
}

extern "C" int dpdf_gated_delta_step(int device, const dpdf_gated_delta_args* args, void* stream) {
    GatedDeltaArgs a;
    if (int rc = gd_check(args, true, a)) return rc;
    if (!args->batch || !args->frames) return DPDF_OK;
    // a head's state is addressed with 32 bits
    if ((long)a.Dk * a.Dv > (1L << 28)) return set_err(DPDF_E_INVALID, "gated delta rule: a head of %d x %d is too large", a.Dk, a.Dv);
    gd_pieces(a, op_bytes(args->dtype));
    a.whole &= a.even && gd_fours(a.v, a.vs, op_bytes(args->dtype));
    OpDevice dev(device);
    HIP_TRY(dev.err);
    a.strips = (a.Dv + 31) / 32;
    const unsigned grid = (unsigned)((long)args->batch * a.Hv * a.strips);
    gd_type(args->dtype, [&](auto t) { gd_launch_step<decltype(t)>(a, grid, (hipStream_t)stream); });
    HIP_TRY(hipGetLastError());
    return DPDF_OK;
}

extern "C" int dpdf_w4_quantize(int device, const dpdf_w4_quantize_args* args, void* stream) {
    if (!args) return set_err(DPDF_E_INVALID, "null argument");
    const dpdf_w4_quantize_args& x = *args;
    if (int rc = w4_check(x.dtype, x.in_dim, x.out_dim, x.group, "w4 quantize")) return rc;
    const long groups = ((long)x.in_dim + x.group - 1) / x.group, bytes = ((long)x.in_dim + 1) / 2;
    if (!x.weight || !x.codes || !x.scales) return set_err(DPDF_E_INVALID, "null argument");
    if (x.weight_stride < 0 || x.codes_pitch < bytes || x.scales_stride < groups || (x.zeros && x.zeros_pitch < groups))
        return set_err(DPDF_E_INVALID, "w4 quantize: rows overlap");
    const int e = op_bytes(x.dtype);
    if (!op_aligned(x.weight, e) || !op_aligned(x.scales, e)) return set_err(DPDF_E_INVALID, "w4 quantize: a pointer is not aligned to its type");
    const long rows = x.out_dim, n[1] = {rows};
    const OpSpan w = op_span(x.weight, &x.weight_stride, n, 1, x.in_dim, e), o[3] = {op_span(x.codes, &x.codes_pitch, n, 1, bytes, 1), op_span(x.scales, &x.scales_stride, n, 1, groups, e),
                     {(const char*)x.zeros, (const char*)x.zeros + (x.zeros ? (rows - 1) * x.zeros_pitch + groups : 0)}};
    for (int i = 0; i < 3; ++i)
        if (op_meet(w, o[i]) || op_meet(o[i], o[(i + 1) % 3])) return set_err(DPDF_E_INVALID, "w4 quantize: an output overlaps another tensor");
    OpDevice dev(device);
    HIP_TRY(dev.err);
    W4QuantArgs a{x.weight, x.weight_stride, x.codes, x.codes_pitch, x.scales, x.scales_stride, x.zeros, x.zeros_pitch, x.out_dim, x.in_dim, x.group, (int)groups};
    const long need = ((long)x.out_dim * groups + 3) / 4, most = OP_THREADS / 256;      // four waves, a group each at a time
    const unsigned grid = (unsigned)(need < most ? need : most);
    if (x.dtype == DPDF_F32) w4_quantize_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else if (x.dtype == DPDF_F16) w4_quantize_kernel<__half><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else w4_quantize_kernel<__hip_bfloat16><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    HIP_TRY(hipGetLastError());
    return DPDF_OK;
}

extern "C" int dpdf_w4_matvec(int device, const dpdf_w4_matvec_args* args, void* stream) {
    if (!args) return set_err(DPDF_E_INVALID, "null argument");
    const dpdf_w4_matvec_args& x = *args;
    if (int rc = w4_check(x.dtype, x.in_dim, x.out_dim, x.group, "w4 matvec")) return rc;
    if (x.scale_dtype != DPDF_F32 && x.scale_dtype != x.dtype) return set_err(DPDF_E_INVALID, "w4 matvec: unsupported dtypes %d / %d", x.dtype, x.scale_dtype);
    if (x.rows < 0) return set_err(DPDF_E_INVALID, "w4 matvec: negative size rows=%d", x.rows);
    if (!x.rows) return DPDF_OK;
    const long groups = ((long)x.in_dim + x.group - 1) / x.group, bytes = ((long)x.in_dim + 1) / 2;
    if (!x.x || !x.codes || !x.scales || !x.out) return set_err(DPDF_E_INVALID, "null argument");
    if (x.x_stride < 0 || x.codes_pitch < 0 || x.scales_stride < 0 || x.zeros_pitch < 0) return set_err(DPDF_E_INVALID, "w4 matvec: negative stride");
    if (x.rows > 1 && x.out_stride < x.out_dim) return set_err(DPDF_E_INVALID, "w4 matvec: elements of out share memory");
    const int e = op_bytes(x.dtype), se = op_bytes(x.scale_dtype);
    if (!op_aligned(x.x, e) || !op_aligned(x.out, e) || !op_aligned(x.bias, e) || !op_aligned(x.scales, se)) return set_err(DPDF_E_INVALID, "w4 matvec: a pointer is not aligned to its type");
    const long rows[1] = {x.rows}, outs[1] = {x.out_dim};
    const OpSpan o = op_span(x.out, &x.out_stride, rows, 1, x.out_dim, e);
    const OpSpan in[5] = {op_span(x.x, &x.x_stride, rows, 1, x.in_dim, e), op_span(x.codes, &x.codes_pitch, outs, 1, bytes, 1), op_span(x.scales, &x.scales_stride, outs, 1, groups, se),
                          {(const char*)x.zeros, (const char*)x.zeros + (x.zeros ? (x.out_dim - 1L) * x.zeros_pitch + groups : 0)}, {(const char*)x.bias, (const char*)x.bias + (x.bias ? (long)x.out_dim * e : 0)}};
    for (const OpSpan& i : in) if (op_meet(o, i)) return set_err(DPDF_E_INVALID, "w4 matvec: out overlaps an input");
    W4Args a{x.x, x.x_stride, x.codes, x.codes_pitch, x.scales, x.scales_stride, x.zeros, x.zeros_pitch, x.bias, x.out, x.out_stride, x.rows, x.in_dim, x.out_dim, x.group, 0};
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess) cus = 256;      // a missing device is reported below
    const W4Split split = w4_split(a, x.dtype, cus);
    const int nt = split.nt;
    a.tiles = (unsigned)((x.out_dim + 16L * nt - 1) / (16 * nt));
    const long grid = a.tiles * ((x.rows + 15L) / 16);
    if (grid > OP_THREADS / (64 * split.nw)) return set_err(DPDF_E_INVALID, "w4 matvec: %d rows are too many for one call", x.rows);
    OpDevice dev(device);
    HIP_TRY(dev.err);
    gd_types(x.dtype, x.scale_dtype, [&](auto t, auto g) { w4_launch<decltype(t), decltype(g)>(a, (unsigned)grid, split, (hipStream_t)stream); });
    HIP_TRY(hipGetLastError());
    return DPDF_OK;
}
