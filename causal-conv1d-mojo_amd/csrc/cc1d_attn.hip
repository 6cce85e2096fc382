// cc1d_attn.hip -- linear attention with a decay for each head: the plan of a
// call (segments, workspace, jobs), and what runs beside its main kernel
// (cc1d_attn_kernels.hpp): the states handed from segment to segment, the
// gradient of the decays, and the sums over heads that share their queries.
#include "cc1d_attn_kernels.hpp"

namespace cc1d {
namespace {

constexpr int64_t kAlign = 4;  // floats

struct Plan {
    int64_t seqs, seg, slots, per_row, states;  // states: between segments
    bool cut() const { return slots > seqs; }
};

// Segments of about `seg` positions, or whole sequences.
Plan cut_of(const cc1d_attn_params& p, int64_t seg) {
    Plan pl;
    pl.seqs = p.cu_seqlens ? p.num_seqs : p.batch;
    constexpr int64_t c = kMaxChunk;
    seg = ceil_div(seg > 0 ? seg : 1, c) * c;
    if (seg >= p.seqlen) {
        pl.seg = seg;
        pl.per_row = 1;
        // (with cu_seqlens a slot starts at cu[i] / seg + i: seg has to be more than the last start)
        if (p.cu_seqlens) pl.seg += c;
        pl.slots = pl.seqs;
        pl.states = 0;
    } else {
        pl.seg = seg;
        pl.per_row = ceil_div(p.seqlen, seg);
        pl.slots = p.cu_seqlens ? p.seqlen / seg + p.num_seqs : p.batch * pl.per_row;
        pl.states = p.cu_seqlens ? (p.seqlen - 1) / seg : p.batch * (pl.per_row - 1);
    }
    return pl;
}

// Positions after which the decays' gradient begins anew from the states (attn_decay_grad_kernel), which the backward
// leaves on the way. In fp32 512: its error over 2048 positions of 48 heads of 64 x 64 is 3.3e-7 to 3.9e-7 of it where
// heads remember 2 to 1000 positions, with 1024 4.1e-7 to 6.8e-7, with 2048 4.9e-7 to 8.6e-7 (1e-7 where they forget
// faster, with any); 4 x 2048, 40 heads of 128 x 128, both directions: 1211, 1209 and 1206 us. 16 bits round far above
// that (2e-4), and their states are larger beside what else is moved: 482, 460 and 448 us for the same in bf16.
int64_t piece_of(const cc1d_attn_params& p) { return p.dtype == CC1D_DTYPE_FP32 ? 512 : 2048; }

// Sequences run as one block per head where those come near to filling the
// chip (256 CUs, two or three blocks each); longer ones are cut into segments
// that run side by side, from states that a first pass over keys and values
// alone provides, which costs about half as much again. Measured, bf16 128 x 128,
// both directions: batch 4 of 40 heads, 2048 positions 450 us whole and 552 in
// three segments (forward alone 151 and 149); fp32 80 x 72, 16 heads of 2048: 248
// us in segments of 192 (this rule's), 193 with 128, 1006 whole. Packed sequences are cut whatever
// their number, as their lengths are not known here and one of them may be nearly
// all: a block's share is then 1 / 768 of the work or 192 positions, whichever
// is more (8192 ragged positions, 32 heads, forward: 166 us, and 188 with segments
// of 256, 183 with 512, 225 whole).
// Below 384 positions two more launches cost more than they save (16 heads of
// 128 x 128, bf16, forward: 256 positions 22 us whole, 30 in two segments; 448: 35
// and 38 in three; 1024: 73 and 43 in six; both directions 71 and 86, 86 and 99,
// 179 and 116).
Plan plan_of(const cc1d_attn_params& p, int jobs) {
    int64_t seg;
    if (p.cu_seqlens) {
        seg = (int64_t)((double)p.seqlen * (double)p.heads / 768.0);
    } else {
        const double blocks = (double)p.batch * (double)p.heads * jobs;
        seg = blocks >= 128.0 ? p.seqlen : (int64_t)((double)p.seqlen * blocks / 512.0);
    }
    if (jobs > 1 && p.dtype == CC1D_DTYPE_FP32 && seg < p.seqlen && seg > piece_of(p)) seg = piece_of(p);  // (16 bits need it less than the states' room)
    return cut_of(p, p.seqlen < 384 ? p.seqlen : seg < 160 ? 160 : seg);
}

// Pieces of the walk over a decay's gradient: where sequences are cut, their segments.
Plan pieces_of(const cc1d_attn_params& p) {
    const Plan pl = plan_of(p, kAttnJobs);
    return pl.cut() ? pl : cut_of(p, piece_of(p));
}

int64_t aligned(int64_t n) { return ceil_div(n, kAlign) * kAlign; }

AttnArgs args_of(const cc1d_attn_params& p, const Plan& pl, int jobs) {
    AttnArgs a{};
    a.g = p.g;
    for (int i = 0; i < 3; ++i) a.g_stride[i] = p.g_stride[i];
    a.cu = p.cu_seqlens;
    a.batch = p.batch;
    a.seqlen = p.seqlen;
    a.num_seqs = pl.seqs;
    a.seg = pl.seg;
    a.heads = (uint32_t)p.heads;
    a.jobs = (uint32_t)jobs;
    a.slots = (uint32_t)pl.slots;
    a.per_row = (uint32_t)pl.per_row;
    a.heads_div = FastDiv(a.heads);
    a.jobs_div = FastDiv(a.jobs);
    a.row_div = FastDiv(a.per_row);
    a.blocks = (uint32_t)(pl.slots * p.heads * jobs);
    return a;
}

AttnOperand operand(const void* ptr, const int64_t (&s)[4], int64_t div) {
    AttnOperand o{ptr, {}, (uint32_t)div};
    for (int i = 0; i < 4; ++i) o.s[i] = s[i];
    return o;
}

// (n, heads, rows, cols) contiguous
AttnState state(float* ptr, int64_t heads, int64_t rows, int64_t cols) { return {ptr, {heads * rows * cols, rows * cols, cols, 1}}; }
AttnState strided(const float* ptr, const int64_t (&s)[4]) { return {const_cast<float*>(ptr), {s[0], s[1], s[2], s[3]}}; }
AttnState turned(AttnState s) {
    const int64_t t = s.s[2];
    s.s[2] = s.s[3];
    s.s[3] = t;
    return s;
}

int launch_jobs(int dtype, const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        return attn_quick<T>(a) ? launch_attn_modes<T, true>(a, da, dc, states, stream) : launch_attn_modes<T, false>(a, da, dc, states, stream);
    });
}

// ---- states from segment to segment

struct CombineArgs {
    AttnArgs a;  // the segments (jobs of the first pass)
    uint32_t pieces;  // of 256 vectors
};

// The first pass left after every segment but a sequence's last what that
// segment adds to a state of 0; afterwards the state itself is there. A thread
// for V values, in the order of memory; the walk over the segments is serial,
// with eight of them on their way. Bound by the states, read and written once
// (170 MB for 8192 positions of 32 heads of 128 x 128 in segments of 384:
// 22 us, from the last-level cache in part).
template <int V> __global__ void __launch_bounds__(256) attn_combine_kernel(const CombineArgs arg) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const AttnArgs& a = arg.a;
    const uint32_t rest = blockIdx.x / arg.pieces, jn = rest / a.heads, h = rest - jn * a.heads;
    const AttnJob& job = a.job[jn];
    const int32_t per = job.da * job.dc, e = (int32_t)((blockIdx.x - rest * arg.pieces) * 256 + threadIdx.x) * V;
    if (e >= per) return;
    const bool turned = job.seg.s[3] != 1;  // rows are next to each other
    const int32_t inner = turned ? job.da : job.dc;
    const float* const decay = job.decay + h;
    for (int64_t seq = blockIdx.y; seq < a.num_seqs; seq += gridDim.y) {
        AttnSpan s;
        if (a.cu == nullptr) {
            s.states = seq * (a.per_row - 1);
            s.len = a.seqlen;
        } else {
            const int64_t first = clamp_pos(a.cu[seq], a.seqlen);
            s.len = clamp_pos(a.cu[seq + 1], a.seqlen) - first;
            s.states = first / a.seg;
        }
        if (s.len <= a.seg) continue;
        s.segs = (s.len + a.seg - 1) / a.seg;
        s.index = 0;
        const int64_t n = s.segs - 1, start = s.after(job.reverse), dir = job.reverse ? -1 : 1;
        vec cur = 0.0f;
        if (job.first.p) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int32_t out = (e + i) / inner, in = (e + i) - out * inner;
                cur[i] = job.first.p[seq * job.first.s[0] + h * job.first.s[1] + (turned ? in : out) * job.first.s[2] + (turned ? out : in) * job.first.s[3]];
            }
        }
        constexpr int K = 8;
        float* at = job.seg.p + start * job.seg.s[0] + h * job.seg.s[1] + e;
        const float* by_at = decay + start * a.heads;
        const int64_t step = dir * job.seg.s[0], by_step = dir * (int64_t)a.heads;
        for (int64_t i = 0; i < n; i += K, at += K * step, by_at += K * by_step) {
            vec adds[K];
            float by[K];
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (i + k < n) {
                    by[k] = by_at[k * by_step];
                    adds[k] = *reinterpret_cast<const vec*>(at + k * step);
                }
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (i + k < n) {
                    cur = by[k] * cur + adds[k];
                    *reinterpret_cast<vec*>(at + k * step) = cur;
                }
        }
    }
}

int run_segments(const cc1d_attn_params& p, const Plan& pl, const AttnArgs& a, int da, int dc, hipStream_t stream) {
    const int st = launch_jobs(p.dtype, a, da, dc, true, stream);
    if (st != CC1D_OK) return st;
    bool whole = (int64_t)da * dc % 4 == 0;
    for (uint32_t j = 0; j < a.jobs; ++j) whole = whole && reinterpret_cast<uintptr_t>(a.job[j].seg.p) % 16 == 0;
    const uint32_t pieces = (uint32_t)ceil_div((int64_t)da * dc, whole ? 1024 : 256);
    const dim3 grid((unsigned)(pieces * p.heads * a.jobs), (unsigned)(pl.seqs < 1024 ? pl.seqs : 1024));
    return launch(whole ? attn_combine_kernel<4> : attn_combine_kernel<1>, grid, dim3(256), stream, CombineArgs{a, pieces});
}

// ---- the gradient of the decays

struct DecayGradArgs {
    const float* row_dots;  // q . (what dq gets from the state before its chunk), (heads, tokens)
    const float* col_dots;  // k . (what dk gets from the gradient of the state after its chunk)
    const float* over;      // the chunk's pairs over each position
    const void* g;
    void* dg;               // (tokens, heads)
    AttnState dfinal;       // gradients of the final states; p null: not used
    const float* tail;      // and the states before the last chunks, as `states`
    int64_t g_stride[3];
    int64_t tokens;
    int32_t dk, dv;
    AttnArgs at;  // the pieces (as a sequence's segments), heads
    // states between pieces, forwards and backwards: (places, heads, dk, dv), dv rounded up to whole vectors where the
    // walks left them (`pitch`); null: one piece a sequence
    const float *states, *grads;
    int32_t pitch;
};

// The sum over a block of 256, in everybody, in a fixed order. (NaN and infinities of one wavefront reach all.)
__device__ __forceinline__ double block_sum_f64(double v, double (&part)[4]) {
    const double s = lane63(wave_prefix_f64(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ double tail_dot(const DecayGradArgs& a, int64_t seq, uint32_t h, double (&part)[4]) {
    if (a.dfinal.p == nullptr) return 0.0;
    const float* const x = a.dfinal.p + seq * a.dfinal.s[0] + h * a.dfinal.s[1];
    const int pitch = (int)kept_rows(a.dv);
    const float* const y = a.tail + (seq * a.at.heads + h) * a.dk * pitch;
    double s = 0.0;
    for (int c = threadIdx.x & 63; c < a.dv; c += 64) {
#pragma unroll 8
        for (int r = threadIdx.x >> 6; r < a.dk; r += 4) s += (double)x[r * a.dfinal.s[2] + c * a.dfinal.s[3]] * (double)y[r * pitch + c];
    }
    return block_sum_f64(s, part);
}

// dg[t] = exp(g[t]) <G[t], S[t-1]>, G the gradient of the state: all that a
// decay carries from the positions before it to itself and the ones behind. By
// chunks, the kernel that forms dq and dk leaves three shares of that, none of
// which holds anything that does not pass over the position:
//     dg[t] = over[t]                      pairs of the chunk, on its two sides
//           + sum of row_dots from t on    out of the chunk's first state
//           + sum of col_dots before t     into the gradient after the chunk
//           + X                            from before the chunk to behind it.
// X is the same for a chunk's positions. With D the whole at a boundary between
// chunks, X = D[end] - sum col_dots and D[start] = X + sum row_dots, from the
// sequence's last chunk on, whose X is exp(its g) <dfinal, S before it>. These
// are differences, and errors of D's size add up from chunk to chunk, as the
// square root of their number: D is formed anew, exp(g) <G, S>, after each
// piece (piece_of()), and X is 0 where the chunk's decay is less than 2^-24, as
// it then is below those errors. What is left is an error of D's size at a
// position that forgets far more than the ones around it.
// (A running sum of q . dq - k . dk alone takes back all that does not pass
// over a position, and where heads forget at once dg is far less than that.
// 2048 positions of 64 x 64, fp32, exp(g) = exp(-4), exp(-10): off by 4e-4 and
// 0.1 of dg, root mean square, this by 1e-7.)
// A block per piece and head walks over 1024 positions at a time, four to a
// thread, GL threads to a chunk, sums in 64 bits. Latency bounds it (14 us for
// 4 x 2048, 40 heads of 128 x 128), and for many short pieces their states.
template <typename T, int GL> __global__ void __launch_bounds__(256) attn_decay_grad_kernel(const DecayGradArgs a) {
    constexpr int K = 4, TILE = 256 * K, NG = 256 / GL;  // positions a thread, of a turn; chunks of a turn
    __shared__ double part[4], rows_of[NG], cols_of[NG];
    __shared__ float passes[NG];
    __shared__ double whole_of;
    const int tid = threadIdx.x, lane = tid & 63, gl = tid % GL, group = tid / GL;
    const int64_t heads = a.at.heads;
    const uint32_t slot = a.at.heads_div.div(blockIdx.x), h = blockIdx.x - slot * a.at.heads;
    const AttnSpan sp = attn_span(a.at, slot);
    if (!sp.live) return;
    const int64_t row = a.at.cu ? 0 : sp.seq;
    const T* const g = static_cast<const T*>(a.g) + row * a.g_stride[0] + h * a.g_stride[2];
    const int64_t begin = sp.first + sp.index * a.at.seg, last = begin + a.at.seg < sp.first + sp.len ? begin + a.at.seg : sp.first + sp.len;
    // D at the piece's end; at the sequence's, <dfinal, S before the last chunk>
    double carry = 0.0;
    const bool tail = sp.index + 1 == sp.segs;
    if (!tail) {
        const float decay = to_f32(g[last * a.g_stride[1]]);
        const int64_t per = (int64_t)a.dk * a.pitch, at = (sp.after(false) * heads + h) * per;
        const float *const x = a.states + at, *const y = a.grads + at;
        double s = 0.0;
#pragma unroll 8
        for (int i = tid; i < (int)per; i += 256) s += (double)x[i] * (double)y[i];
        s = block_sum_f64(s, part);
        carry = decay < kNoDecay ? 0.0 : exp((double)decay) * s;
    } else {
        carry = tail_dot(a, sp.seq, h, part);
    }
    const int64_t base = row * a.at.seqlen;
    T* const dg = static_cast<T*>(a.dg);
    bool first = true;
    const int last_group = (int)((last - begin - 1) % TILE) / (K * GL);  // of the first turn
    for (int64_t from = begin + (last - begin - 1) / TILE * TILE; from >= begin && from < last; from -= TILE) {
        // thread t has positions from + K t + i
        double u[K], v[K], us = 0.0, vs = 0.0, gs = 0.0;
        float w[K], decay[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int64_t t = from + K * tid + i, at = h * a.tokens + base + t;
            const bool in = t < last;
            u[i] = in ? (double)a.row_dots[at] : 0.0;
            v[i] = in ? (double)a.col_dots[at] : 0.0;
            w[i] = in ? a.over[at] : 0.0f;
            decay[i] = in ? to_f32(g[t * a.g_stride[1]]) : 0.0f;
            us += u[i];
            vs += v[i];
            gs += log_decay(decay[i]);
        }
        // rows from this thread's on, columns up to its, the decays of the chunk. (No difference of sums: one that is
        // not finite stays on its side.)
#pragma unroll
        for (int d = 1; d < GL; d *= 2) {
            const double later = __shfl_down(us, d, GL), earlier = __shfl_up(vs, d, GL);
            if (gl + d < GL) us += later;
            if (gl >= d) vs += earlier;
            gs += __shfl_xor(gs, d);
        }
        const double later = __shfl_down(us, 1, GL), earlier = __shfl_up(vs, 1, GL);
        double behind = gl + 1 < GL ? later : 0.0, before = gl > 0 ? earlier : 0.0;
        __syncthreads();  // (of the turn before)
        if (gl == 0) rows_of[group] = us;
        if (gl == GL - 1) {
            cols_of[group] = vs;
            passes[group] = gs < -24.0 * 0.6931471805599453 ? 0.0f : 1.0f;
            if (first && tail && group == last_group) {
                passes[group] = 0.0f;
                whole_of = carry == 0.0 ? 0.0 : exp(gs) * carry;
            }
        }
        __syncthreads();
        // D at a chunk's start is p D[end] + (rows - p cols): a lane a chunk, from the last one back
        const int n = lane % NG;
        const double rows = rows_of[n], cols = cols_of[n], p = (double)passes[n], own = first && tail && n == last_group ? whole_of : 0.0;
        double all = p, add = own + (rows - p * cols);
#pragma unroll
        for (int d = 1; d < NG; d *= 2) {
            const double all_later = __shfl_down(all, d, NG), add_later = __shfl_down(add, d, NG);
            if (n + d < NG) {
                add += all * add_later;
                all *= all_later;
            }
        }
        const double start = add + all * carry, next = __shfl_down(start, 1, NG);
        const double x = __shfl(own + p * ((n + 1 < NG ? next : carry) - cols), group);
        carry = __shfl(start, 0);
        first = false;
        double lower[K];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            lower[i] = before;
            before += v[i];
        }
#pragma unroll
        for (int i = K - 1; i >= 0; --i) {
            const int64_t t = from + K * tid + i;
            behind += u[i];
            // nothing is carried over a decay of 0
            if (t < last) dg[(base + t) * heads + h] = from_f32<T>(decay[i] < kNoDecay ? 0.0f : (float)(((double)w[i] + x) + (lower[i] + behind)));
        }
    }
    if (a.at.cu) {
        if (sp.seq == 0 && sp.index == 0)
            for (int64_t t = tid; t < sp.first; t += 256) dg[t * heads + h] = from_f32<T>(0.0f);
        if (sp.seq == a.at.num_seqs - 1 && sp.index + 1 == sp.segs)
            for (int64_t t = last + tid; t < a.at.seqlen; t += 256) dg[t * heads + h] = from_f32<T>(0.0f);
    }
}

// ---- sums over the heads that share a key head

struct GroupSumArgs {
    const float* part[2];  // (tokens, heads, dk)
    void* out[2];          // (tokens, key_heads, dk)
    int64_t n;             // values of out
    int32_t each, dk;      // heads to a key head
};

// A thread for V neighbours; each value is read and written once.
template <typename T, int V> __global__ void __launch_bounds__(256) attn_group_sum_kernel(const GroupSumArgs a) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const float* const part = a.part[blockIdx.y];
    T* const out = static_cast<T*>(a.out[blockIdx.y]);
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < a.n; i += (int64_t)gridDim.x * 256 * V) {
        const float* const at = part + i / a.dk * (a.each - 1) * a.dk + i;
        vec s = 0.0f;
#pragma unroll 4
        for (int r = 0; r < a.each; ++r) s += *reinterpret_cast<const vec*>(at + (int64_t)r * a.dk);
        T w[V];
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = from_f32<T>(s[e]);
        __builtin_memcpy(__builtin_assume_aligned(out + i, V * sizeof(T)), w, sizeof(w));
    }
}

// The backward's workspace, in floats.
struct Room {
    int64_t dots, part, between, decay, tail, total;
};
Room room_of(const cc1d_attn_bwd_params& b, const Plan& pl) {
    const cc1d_attn_params& p = b.fwd;
    const int64_t tokens = p.batch * p.seqlen, per = p.heads * p.dk * p.dv;
    Room r;
    r.dots = aligned(tokens * p.heads);
    r.part = p.heads == p.key_heads ? 0 : aligned(tokens * p.heads * p.dk);
    r.between = aligned(pieces_of(p).states * (pl.cut() ? per : p.heads * p.dk * kept_rows(p.dv)));
    r.decay = aligned(pl.states * p.heads);
    r.tail = b.dfinal_states ? aligned(pl.seqs * p.heads * p.dk * kept_rows(p.dv)) : 0;
    r.total = 3 * r.dots + 2 * r.part + 2 * r.between + 2 * r.decay + r.tail;
    return r;
}

}  // namespace

bool attn_fits(const cc1d_attn_params& p) {
    // inside a state, and from row to row of a chunk of outputs, the kernels count in 32 bits; so do launches:
    // blocks of 256 threads, 32-bit thread counts: one a slot, head and job, or one a piece of 256 values of a state
    const double seqs = p.cu_seqlens ? (double)p.num_seqs : (double)p.batch;
    if ((double)p.heads >= (double)(1 << 15) || seqs * (double)p.heads * kAttnJobs >= (double)(1 << 23)) return false;
    if ((double)p.batch * (double)p.seqlen >= (double)((int64_t)1 << 40) || p.seqlen >= ((int64_t)1 << 31) - 4096) return false;
    return (double)plan_of(p, kAttnJobs).slots * (double)p.heads * kAttnJobs < (double)(1 << 24) &&
           (double)plan_of(p, 1).slots * (double)p.heads < (double)(1 << 24) &&
           (double)pieces_of(p).slots * (double)p.heads < (double)(1 << 24) && (double)p.heads * 2 * 64 < (double)(1 << 24);
}

int64_t attn_workspace_floats(const cc1d_attn_params& p) {
    const Plan pl = plan_of(p, 1);
    return aligned(pl.states * p.heads * p.dk * p.dv) + aligned(pl.states * p.heads);
}

int launch_attn_fwd(const cc1d_attn_params& p, hipStream_t stream) {
    const Plan pl = plan_of(p, 1);
    const int64_t per = p.heads / p.key_heads;
    AttnArgs a = args_of(p, pl, 1);
    AttnJob& j = a.job[0];
    j.a = operand(p.q, p.q_stride, per);
    j.b = operand(p.k, p.k_stride, per);
    j.c = operand(p.v, p.v_stride, 1);
    j.first = strided(p.initial_states, p.initial_states_stride);
    j.last = state(p.final_states, p.heads, p.dk, p.dv);
    j.out = p.out;
    j.da = (int32_t)p.dk;
    j.dc = (int32_t)p.dv;
    j.p_scale = j.in_scale = (float)p.scale;
    j.w_scale = 1.0f;
    if (pl.cut()) {
        j.seg = state(p.workspace, p.heads, p.dk, p.dv);
        j.decay = p.workspace + aligned(pl.states * p.heads * p.dk * p.dv);
        const int st = run_segments(p, pl, a, (int)p.dk, (int)p.dv, stream);
        if (st != CC1D_OK) return st;
    }
    return launch_jobs(p.dtype, a, (int)p.dk, (int)p.dv, false, stream);
}

int64_t attn_bwd_workspace_floats(const cc1d_attn_bwd_params& b) { return room_of(b, plan_of(b.fwd, kAttnJobs)).total; }

int launch_attn_bwd(const cc1d_attn_bwd_params& b, hipStream_t stream) {
    const cc1d_attn_params& p = b.fwd;
    const Plan pl = plan_of(p, kAttnJobs);
    const Room room = room_of(b, pl);
    const int64_t per = p.heads / p.key_heads, tokens = p.batch * p.seqlen;
    const int dk = (int)p.dk, dv = (int)p.dv;
    const bool shared = per > 1;
    float* ws = b.workspace;
    auto take = [&ws](int64_t n) {
        float* at = n ? ws : nullptr;
        ws += n;
        return at;
    };
    float *const row_dots = take(room.dots), *const col_dots = take(room.dots), *const over = take(room.dots);
    float *const dq_part = take(room.part), *const dk_part = take(room.part);
    float *const states = take(room.between), *const grads = take(room.between);
    float *const decay_s = take(room.decay), *const decay_g = take(room.decay);
    float* const tail = take(room.tail);

    const AttnOperand q = operand(p.q, p.q_stride, per), k = operand(p.k, p.k_stride, per), v = operand(p.v, p.v_stride, 1);
    const AttnOperand d = operand(b.dout, b.dout_stride, 1);
    const AttnState first = strided(p.initial_states, p.initial_states_stride);
    const AttnState last_grad = strided(b.dfinal_states, b.dfinal_states_stride);
    const float scale = (float)p.scale;

    AttnJob jq{}, jk{}, jv{};
    jq.a = d; jq.b = v; jq.c = k; jq.x = q;
    jq.first = turned(first);
    jq.tail = tail;
    jq.seg = turned(state(states, p.heads, dk, dv));
    jq.decay = decay_s;
    jq.out = shared ? dq_part : b.dq;
    jq.dots = row_dots;
    jq.da = dv; jq.dc = dk;
    jq.p_scale = jq.in_scale = scale; jq.w_scale = 1.0f;
    jq.out_f32 = shared;

    jk.a = v; jk.b = d; jk.c = q; jk.x = k;
    jk.first = turned(last_grad);
    jk.seg = turned(state(grads, p.heads, dk, dv));
    jk.decay = decay_g;
    jk.out = shared ? dk_part : b.dk;
    jk.dots = col_dots;
    jk.da = dv; jk.dc = dk;
    jk.p_scale = jk.w_scale = scale; jk.in_scale = 1.0f;
    jk.reverse = 1;
    jk.out_f32 = shared;

    jv.a = k; jv.b = q; jv.c = d; jv.x = v;
    jv.first = last_grad;
    jv.last = state(b.dinitial_states, p.heads, dk, dv);
    jv.seg = state(grads, p.heads, dk, dv);
    jv.decay = decay_g;
    jv.out = b.dv;
    jv.over = over;
    jv.da = dk; jv.dc = dv;
    jv.p_scale = jv.w_scale = scale; jv.in_scale = 1.0f;
    jv.reverse = 1;

    if (pl.cut()) {
        // both states as (dk, dv): K^T V forwards, Q^T dO backwards
        AttnArgs s = args_of(p, pl, 2);
        s.job[0] = jv;
        s.job[0].b = k; s.job[0].c = v;
        s.job[0].first = first;
        s.job[0].seg = state(states, p.heads, dk, dv);
        s.job[0].decay = decay_s;
        s.job[0].w_scale = 1.0f;
        s.job[0].reverse = 0;
        s.job[1] = jv;
        const int st = run_segments(p, pl, s, dk, dv, stream);
        if (st != CC1D_OK) return st;
    }
    // where sequences are not cut, the walks leave states for the decays' gradient as they go
    const Plan pieces = pieces_of(p);
    if (!pl.cut() && pieces.cut()) {
        jq.mark = states;
        jk.mark = grads;
        jq.piece = jk.piece = pieces.seg;
        jq.pieces = jk.pieces = pieces.per_row;
    }
    int st;
    const bool alike = (dk <= 64) == (dv <= 64);  // one kernel for all
    if (alike) {
        AttnArgs a = args_of(p, pl, 3);
        a.job[0] = jq; a.job[1] = jk; a.job[2] = jv;
        st = launch_jobs(p.dtype, a, dk, dv, false, stream);
    } else {
        AttnArgs a = args_of(p, pl, 2);
        a.job[0] = jq; a.job[1] = jk;
        st = launch_jobs(p.dtype, a, dv, dk, false, stream);
        if (st != CC1D_OK) return st;
        AttnArgs c = args_of(p, pl, 1);
        c.job[0] = jv;
        st = launch_jobs(p.dtype, c, dk, dv, false, stream);
    }
    if (st != CC1D_OK) return st;
    if (tokens == 0) return CC1D_OK;
    DecayGradArgs dg{row_dots, col_dots, over, p.g, b.dg, last_grad, tail, {}, tokens, dk, dv, args_of(p, pieces, 1), states, grads, (int32_t)(pl.cut() ? dv : kept_rows(dv))};
    for (int i = 0; i < 3; ++i) dg.g_stride[i] = p.g_stride[i];
    st = with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        static_assert(chunk_of<T>(64, 128) == chunk_of<T>(128, 64), "dq, dk and dv in the same chunks");
        constexpr int least = chunk_of<T>(128, 128), most = chunk_of<T>(64, 64);
        const bool wide = chunk_of<T>(attn_dim_of(dv), attn_dim_of(dk)) == most;
        return launch(wide ? attn_decay_grad_kernel<T, most / 4> : attn_decay_grad_kernel<T, least / 4>, dim3(dg.at.blocks), dim3(256), stream, dg);
    });
    if (st != CC1D_OK || !shared) return st;
    const GroupSumArgs gs{{dq_part, dk_part}, {b.dq, b.dk}, tokens * p.key_heads * p.dk, (int32_t)per, dk};
    auto whole = [](const void* at, size_t bytes) { return reinterpret_cast<uintptr_t>(at) % bytes == 0; };
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        const bool four = dk % 4 == 0 && whole(dq_part, 16) && whole(dk_part, 16) && whole(b.dq, 4 * sizeof(T)) && whole(b.dk, 4 * sizeof(T));
        const int64_t blocks = ceil_div(gs.n, four ? 1024 : 256);
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536), 2);
        return launch(four ? attn_group_sum_kernel<T, 4> : attn_group_sum_kernel<T, 1>, grid, dim3(256), stream, gs);
    });
}

}  // namespace cc1d
