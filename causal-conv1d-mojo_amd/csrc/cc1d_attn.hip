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

// Sequences run as one block per head where those come near to filling the
// chip (256 CUs, two or three blocks each); longer ones are cut into segments
// that run side by side, from states that a first pass over keys and values
// alone provides, which costs about half as much again. Measured, bf16 128 x 128,
// both directions: batch 4 of 40 heads, 2048 positions 506 us whole and 602 in
// three segments; fp32 80 x 72, 16 heads of 2048: 242 us in segments of 256,
// about 205 with 128, 933 whole. Packed sequences are cut whatever their
// number, as their lengths are not known here and one of them may be nearly
// all: a block's share is then 1 / 768 of the work or 192 positions, whichever
// is more (8192 positions, 32 heads: 180 us, and 211 with segments of 256, 196
// with 512, 264 whole).
// Below 384 positions two more launches cost more than they save (16 heads of
// 128 x 128, bf16, 256 positions: 22 us whole, 34 in two segments; 448: 40 and
// 37 in three; 1024: 81 and 42 in six).
Plan plan_of(const cc1d_attn_params& p, int jobs) {
    int64_t seg;
    if (p.cu_seqlens) {
        seg = (int64_t)((double)p.seqlen * (double)p.heads / 768.0);
    } else {
        const double blocks = (double)p.batch * (double)p.heads * jobs;
        seg = blocks >= 128.0 ? p.seqlen : (int64_t)((double)p.seqlen * blocks / 512.0);
    }
    return cut_of(p, p.seqlen < 384 ? p.seqlen : seg < 160 ? 160 : seg);
}

// Pieces of the walk over a decay's gradient.
constexpr int64_t kPiece = 4096;
Plan pieces_of(const cc1d_attn_params& p) { return cut_of(p, p.seqlen > 2 * kPiece ? kPiece : p.seqlen); }

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
    const float* row_dots;  // q . dq, (heads, tokens)
    const float* col_dots;  // k . dk
    const void* g;
    void* dg;               // (tokens, heads)
    AttnState dfinal, fin;  // p null: the final states are not used
    int64_t g_stride[3];
    int64_t tokens;
    int32_t dk, dv;
    AttnArgs at;  // the pieces (as a sequence's segments), heads
    // states between segments, forwards and backwards; null: not cut
    const float *seg_s, *seg_g;
    float* sums;  // of pieces and final states, two floats a double: (slots + sequences, heads); null: one piece a sequence
};

typedef uint32_t double_bits __attribute__((ext_vector_type(2), aligned(4)));

// The sum over a block of 256, in everybody, in a fixed order. (NaN and infinities of one wavefront reach all.)
__device__ __forceinline__ double block_sum_f64(double v, double (&part)[4]) {
    const double s = lane63(wave_prefix_f64(v));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ double final_states_dot(const DecayGradArgs& a, int64_t seq, uint32_t h, double (&part)[4]) {
    if (a.dfinal.p == nullptr) return 0.0;
    const float* x = a.dfinal.p + seq * a.dfinal.s[0] + h * a.dfinal.s[1];
    const float* y = a.fin.p + seq * a.fin.s[0] + h * a.fin.s[1];
    double s = 0.0;
    for (int i0 = threadIdx.x; i0 < a.dk * a.dv; i0 += 8 * 256) {  // eight loads of each on their way
        float xs[8], ys[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + 256 * k, r = i / a.dv, c = i - r * a.dv;
            xs[k] = ys[k] = 0.0f;
            if (i < a.dk * a.dv) {
                xs[k] = x[r * a.dfinal.s[2] + c * a.dfinal.s[3]];
                ys[k] = y[r * a.fin.s[2] + c * a.fin.s[3]];
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)xs[k] * (double)ys[k];
    }
    return block_sum_f64(s, part);
}

// Each piece's sum, and by the block of a sequence's last one <G, S> after it.
__global__ void __launch_bounds__(256) attn_dots_sum_kernel(const DecayGradArgs a) {
    __shared__ double part[4];
    const uint32_t slot = a.at.heads_div.div(blockIdx.x), h = blockIdx.x - slot * a.at.heads;
    const AttnSpan sp = attn_span(a.at, slot);
    if (!sp.live) return;
    const int64_t base = h * a.tokens + (a.at.cu ? 0 : sp.seq * a.at.seqlen) + sp.first;
    const int64_t begin = sp.index * a.at.seg, end = begin + a.at.seg < sp.len ? begin + a.at.seg : sp.len;
    double s = 0.0;
    for (int64_t t = begin + threadIdx.x; t < end; t += 256) s += (double)a.row_dots[base + t] - (double)a.col_dots[base + t];
    s = block_sum_f64(s, part);
    double_bits* const sums = reinterpret_cast<double_bits*>(a.sums);
    if (threadIdx.x == 0) sums[(int64_t)slot * a.at.heads + h] = __builtin_bit_cast(u32x2, s);
    if (sp.index + 1 != sp.segs) return;
    s = final_states_dot(a, sp.seq, h, part);
    if (threadIdx.x == 0) sums[((int64_t)a.at.slots + sp.seq) * a.at.heads + h] = __builtin_bit_cast(u32x2, s);
}

// dg[t] = <G, S> after the sequence's last position + sum over s >= t of
// (q . dq - k . dk)[s]: a position's decay carries all that is written before
// it and read from it on, and what is written and read on one side cancels.
// The sums run in 64 bits, but of values that are fp32 products' sums, whose
// errors add up over a walk: where sequences are cut, each segment's begins
// anew from the states at its end, exp(g) <G, S> (16 heads of 80 x 72, 2048
// positions, fp32: off by 2e-7 to 3e-7; 2 x 2048 of 40 heads, uncut, 5e-7 to 7e-7).
// A block per sequence and head walks from the last position to the first, 2 us
// for 1024 of them; uncut sequences of more than 2 kPiece positions go by
// pieces, from their sums (1048576 positions of one
// head: 2033 us as one walk, 23 in pieces).
template <typename T> __global__ void __launch_bounds__(256) attn_decay_grad_kernel(const DecayGradArgs a) {
    __shared__ double part[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int64_t heads = a.at.heads;
    const uint32_t slot = a.at.heads_div.div(blockIdx.x), h = blockIdx.x - slot * a.at.heads;
    const AttnSpan sp = attn_span(a.at, slot);
    if (!sp.live) return;
    const int64_t row = a.at.cu ? 0 : sp.seq;
    const T* const g = static_cast<const T*>(a.g) + row * a.g_stride[0] + h * a.g_stride[2];
    const int64_t begin = sp.first + sp.index * a.at.seg, last = begin + a.at.seg < sp.first + sp.len ? begin + a.at.seg : sp.first + sp.len;
    double carry = 0.0;
    if (a.seg_s != nullptr && sp.index + 1 < sp.segs) {
        // the gradient at the next segment's first position
        const float decay = to_f32(g[last * a.g_stride[1]]);
        const int64_t per = (int64_t)a.dk * a.dv;
        const int64_t at = (sp.after(false) * heads + h) * per;
        const float *const x = a.seg_s + at, *const y = a.seg_g + at;
        double s = 0.0;
#pragma unroll 8
        for (int i = tid; i < (int)per; i += 256) s += (double)x[i] * (double)y[i];
        s = block_sum_f64(s, part);
        carry = decay < -1e5f ? 0.0 : exp((double)decay) * s;
    } else if (a.sums == nullptr) {
        carry = final_states_dot(a, sp.seq, h, part);
    } else {
        const double_bits* const sums = reinterpret_cast<const double_bits*>(a.sums);
        auto sum = [&](int64_t i) { return __builtin_bit_cast(double, (u32x2)sums[i * heads + h]); };
        for (int64_t i = sp.index + 1 + tid; i < sp.segs; i += 256) carry += sum(sp.slot + i);
        carry = block_sum_f64(carry, part) + sum((int64_t)a.at.slots + sp.seq);
    }
    const int64_t base = row * a.at.seqlen;
    T* const dg = static_cast<T*>(a.dg);
    constexpr int K = 4;  // positions a thread
    for (int64_t end = last; end > begin; end -= 256 * K) {
        // thread t has positions end - 1 - K t - i
        double v[K], sum = 0.0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int64_t t = end - 1 - K * tid - i;
            if (t >= begin) {
                const int64_t at = h * a.tokens + base + t;
                sum += (double)a.row_dots[at] - (double)a.col_dots[at];
            }
            v[i] = sum;
        }
        const double incl = wave_prefix_f64(sum);
        __syncthreads();
        if (lane == 63) part[wave] = incl;
        __syncthreads();
        const double later = __shfl_up(incl, 1);  // (not incl - sum, where one that is not finite would reach later positions)
        double before = carry + (lane ? later : 0.0);
        for (int w = 0; w < wave; ++w) before += part[w];
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int64_t t = end - 1 - K * tid - i;
            // nothing is carried over a decay of 0
            if (t >= begin) dg[(base + t) * heads + h] = from_f32<T>(to_f32(g[t * a.g_stride[1]]) < -1e5f ? 0.0f : (float)(before + v[i]));
        }
        carry += (part[0] + part[1]) + (part[2] + part[3]);
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
    int64_t dots, part, seg, decay, fin, sums, total;
};
Room room_of(const cc1d_attn_bwd_params& b, const Plan& pl) {
    const cc1d_attn_params& p = b.fwd;
    const int64_t tokens = p.batch * p.seqlen, per = p.heads * p.dk * p.dv;
    Room r;
    r.dots = aligned(tokens * p.heads);
    r.part = p.heads == p.key_heads ? 0 : aligned(tokens * p.heads * p.dk);
    r.seg = aligned(pl.states * per);
    r.decay = aligned(pl.states * p.heads);
    r.fin = b.dfinal_states ? aligned(pl.seqs * per) : 0;
    const Plan pieces = pieces_of(p);
    r.sums = !pl.cut() && pieces.cut() ? aligned(2 * (pieces.slots + pieces.seqs) * p.heads) : 0;
    r.total = r.sums + 2 * r.dots + 2 * r.part + 2 * r.seg + 2 * r.decay + r.fin;
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
    float *const row_dots = take(room.dots), *const col_dots = take(room.dots);
    float *const dq_part = take(room.part), *const dk_part = take(room.part);
    float *const seg_s = take(room.seg), *const seg_g = take(room.seg);
    float *const decay_s = take(room.decay), *const decay_g = take(room.decay);
    float *const fin = take(room.fin), *const sums = take(room.sums);

    const AttnOperand q = operand(p.q, p.q_stride, per), k = operand(p.k, p.k_stride, per), v = operand(p.v, p.v_stride, 1);
    const AttnOperand d = operand(b.dout, b.dout_stride, 1);
    const AttnState first = strided(p.initial_states, p.initial_states_stride);
    const AttnState last_grad = strided(b.dfinal_states, b.dfinal_states_stride);
    const float scale = (float)p.scale;

    AttnJob jq{}, jk{}, jv{};
    jq.a = d; jq.b = v; jq.c = k; jq.x = q;
    jq.first = turned(first);
    jq.last = turned(state(fin, p.heads, dk, dv));
    jq.seg = turned(state(seg_s, p.heads, dk, dv));
    jq.decay = decay_s;
    jq.out = shared ? dq_part : b.dq;
    jq.dots = row_dots;
    jq.da = dv; jq.dc = dk;
    jq.p_scale = jq.in_scale = scale; jq.w_scale = 1.0f;
    jq.out_f32 = shared;

    jk.a = v; jk.b = d; jk.c = q; jk.x = k;
    jk.first = turned(last_grad);
    jk.seg = turned(state(seg_g, p.heads, dk, dv));
    jk.decay = decay_g;
    jk.out = shared ? dk_part : b.dk;
    jk.dots = col_dots;
    jk.da = dv; jk.dc = dk;
    jk.p_scale = jk.w_scale = scale; jk.in_scale = 1.0f;
    jk.reverse = 1;
    jk.out_f32 = shared;

    jv.a = k; jv.b = q; jv.c = d;
    jv.first = last_grad;
    jv.last = state(b.dinitial_states, p.heads, dk, dv);
    jv.seg = state(seg_g, p.heads, dk, dv);
    jv.decay = decay_g;
    jv.out = b.dv;
    jv.da = dk; jv.dc = dv;
    jv.p_scale = jv.w_scale = scale; jv.in_scale = 1.0f;
    jv.reverse = 1;

    if (pl.cut()) {
        // both states as (dk, dv): K^T V forwards, Q^T dO backwards
        AttnArgs s = args_of(p, pl, 2);
        s.job[0] = jv;
        s.job[0].b = k; s.job[0].c = v;
        s.job[0].first = first;
        s.job[0].seg = state(seg_s, p.heads, dk, dv);
        s.job[0].decay = decay_s;
        s.job[0].w_scale = 1.0f;
        s.job[0].reverse = 0;
        s.job[1] = jv;
        const int st = run_segments(p, pl, s, dk, dv, stream);
        if (st != CC1D_OK) return st;
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
    const Plan walk = pl.cut() ? pl : pieces_of(p);
    DecayGradArgs dg{row_dots, col_dots, p.g, b.dg, last_grad, state(fin, p.heads, dk, dv), {}, tokens, dk, dv, args_of(p, walk, 1), seg_s, seg_g, sums};
    for (int i = 0; i < 3; ++i) dg.g_stride[i] = p.g_stride[i];
    if (sums != nullptr) {
        st = launch(attn_dots_sum_kernel, dim3(dg.at.blocks), dim3(256), stream, dg);
        if (st != CC1D_OK) return st;
    }
    st = with_dtype(p.dtype, [&](auto t) {
        return launch(attn_decay_grad_kernel<decltype(t)>, dim3(dg.at.blocks), dim3(256), stream, dg);
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
