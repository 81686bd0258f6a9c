// qw_op_kv_append on the host, in buffers that end where a page without access begins.  Arguments: heads kv_heads head_dim rows
// mode in_dtype dtype rope fused page in_place.  Ragged sequences, the last row of the buffers the last of a sequence; results
// against the definition in 64 bits (tolerances: a norm within 2^-18, four roundings of fp32, one of bf16).
#include <sys/mman.h>
#include <unistd.h>
#include <string>

#include "common_b200/csrc/qw_kv_append.cu"

namespace qw {
static std::string host_error;
qw_status op_fail(qw_status s, const std::string &msg) { host_error = msg; return s; }
}  // namespace qw

static char *ending(size_t bytes) {  // a buffer of these bytes, its end the end of the last page that may be touched
    const size_t page = sysconf(_SC_PAGESIZE), room = (bytes + page - 1) / page * page;
    char *p = (char *)mmap(nullptr, room + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    if (p == MAP_FAILED || mprotect(p + page, room, PROT_READ | PROT_WRITE)) abort();
    return p + page + room - bytes;
}
static uint32_t state = 1;
static float normal() {
    float s = 0;
    for (int i = 0; i < 4; i++) {
        state = state * 1664525u + 1013904223u;
        s += (float)(state >> 8) / (float)(1 << 24) - 0.5f;
    }
    return 2.f * s;
}

struct Numbers {
    bool bf16;
    char *p;
    Numbers(size_t n, int dtype) : bf16(dtype == QW_DTYPE_BF16), p(ending(n * (bf16 ? 2 : 4))) {
        for (size_t i = 0; i < n; i++) set(i, normal());
    }
    void set(size_t i, float v) {
        if (bf16) ((uint16_t *)p)[i] = host_bf16(v);
        else ((float *)p)[i] = v;
    }
    double operator[](size_t i) const { return bf16 ? __uint_as_float((uint32_t)((uint16_t *)p)[i] << 16) : ((float *)p)[i]; }
    Numbers part(size_t from) const { Numbers r = *this; r.p += from * (bf16 ? 2 : 4); return r; }
};

int main(int argc, char **argv) {
    if (argc != 12) return 2;
    int arg[11];
    for (int i = 0; i < 11; i++) arg[i] = atoi(argv[i + 1]);
    const int H = arg[0], Hkv = arg[1], d = arg[2], rows = arg[3], mode = arg[4], in = arg[5], out = arg[6];
    const bool turned = arg[7], fused = arg[8], in_place = arg[10];
    const int ps = arg[9], half = d / 2, wq = H * d, wk = Hkv * d, rope_len = 600;

    // sequences of many rows and of one; the second stands on rows that are none, the third has no page 1
    std::vector<int> start{0}, len;
    for (int b = 0; start.back() < rows; b++) {
        int n = b % 3 == 1 ? 1 : 37 + 61 * b % 400;
        if (n > rows - start.back()) n = rows - start.back();
        start.push_back(start.back() + n);
        len.push_back(b == 1 ? 0 : b == 3 ? n / 2 : n + 50 * b % 150);
    }
    const int batch = (int)len.size(), max_pages = (800 + ps - 1) / ps, pages = batch * max_pages;
    int *row_start = (int *)ending((batch + 1) * 4), *kv_len = (int *)ending(batch * 4);
    int *table = (int *)ending((size_t)pages * 4);
    memcpy(row_start, start.data(), (batch + 1) * 4);
    memcpy(kv_len, len.data(), batch * 4);
    for (int i = 0; i < pages; i++) table[i] = pages - 1 - i;
    if (batch > 2) table[2 * max_pages + 1] = -1;

    const int ld = fused ? wq + 2 * wk : 0;
    Numbers q((size_t)rows * (fused ? ld : wq), in), k = fused ? q.part(wq) : Numbers((size_t)rows * wk, in);
    Numbers v = fused ? q.part(wq + wk) : Numbers((size_t)rows * wk, in);
    const int lq = fused ? ld : wq, lk = fused ? ld : wk;
    const size_t cells = (size_t)pages * Hkv * ps * d;
    Numbers kc(cells, out), vc(cells, out), qo(in_place ? 1 : (size_t)rows * wq, out);
    Numbers qn(mode == QW_QKNORM_VECTOR ? wq : d, QW_DTYPE_F32), kn(mode == QW_QKNORM_VECTOR ? wk : d, QW_DTYPE_F32);
    Numbers rope((size_t)rope_len * d, QW_DTYPE_F32);
    for (int p = 0; p < rope_len; p++)
        for (int i = 0; i < half; i++) {
            rope.set((size_t)p * d + 2 * i, (float)cos(p * pow(1e4, -i * 2.0 / d)));
            rope.set((size_t)p * d + 2 * i + 1, (float)sin(p * pow(1e4, -i * 2.0 / d)));
        }

    // what is expected, and how far off it may be
    std::vector<double> want_q((size_t)rows * wq), far_q(want_q.size(), 0), want_k(cells), far_k(cells, 0), want_v(cells), far_v(cells, 0);
    for (size_t i = 0; i < cells; i++) { want_k[i] = kc[i]; want_v[i] = vc[i]; }
    const double step = out == QW_DTYPE_BF16 ? 1.0 / 256 : 1.0 / (1 << 24);
    const bool same = mode == QW_QKNORM_NONE && !turned;
    for (int b = 0; b < batch; b++)
        for (int r = start[b]; r < start[b + 1]; r++) {
            const int pos = len[b] - (start[b + 1] - r);
            if (pos < 0 || (turned && pos >= rope_len)) continue;
            const int page = table[b * max_pages + pos / ps];
            for (int h = 0; h < H + 2 * Hkv; h++) {
                const bool isq = h < H, isv = h >= H + Hkv;
                const Numbers &from = isq ? q : isv ? v : k, &w = isq ? qn : kn;
                const int hh = isq ? h : isv ? h - H - Hkv : h - H, l = isq ? lq : lk, heads = isq ? H : Hkv;
                const size_t at = (size_t)r * l + hh * d;
                double n = 1, sum = 0;
                if (!isv && mode != QW_QKNORM_NONE) {
                    const int wide = mode == QW_QKNORM_VECTOR ? heads * d : d;
                    const size_t first = mode == QW_QKNORM_VECTOR ? (size_t)r * l : at;
                    for (int i = 0; i < wide; i++) sum += from[first + i] * from[first + i];
                    n = 1 / sqrt(sum / wide + 1e-6);
                }
                for (int i = 0; i < half; i++) {
                    const int wat = mode == QW_QKNORM_VECTOR ? hh * d : 0;
                    const bool scaled = !isv && mode != QW_QKNORM_NONE;
                    const double x = from[at + i] * (scaled ? n * w[wat + i] : 1), y = from[at + half + i] * (scaled ? n * w[wat + half + i] : 1);
                    const double c = turned && !isv ? rope[(size_t)pos * d + 2 * i] : 1, s = turned && !isv ? rope[(size_t)pos * d + 2 * i + 1] : 0;
                    const double result[2] = {x * c - y * s, y * c + x * s};
                    for (int e = 0; e < 2; e++) {
                        const double far = step * fabs(result[e]) + (isv || same ? 0 : 1.01 * (fabs(x) + fabs(y)) / (1 << 17));
                        if (isq) {
                            want_q[(size_t)r * wq + hh * d + e * half + i] = result[e];
                            far_q[(size_t)r * wq + hh * d + e * half + i] = far;
                        } else if (page >= 0) {
                            const size_t cell = (((size_t)page * Hkv + hh) * ps + pos % ps) * d + e * half + i;
                            (isv ? want_v : want_k)[cell] = result[e];
                            (isv ? far_v : far_k)[cell] = far;
                        }
                    }
                }
            }
        }

    qw_kv_append_args a{};
    a.q = q.p; a.k = k.p; a.v = v.p; a.k_cache = kc.p; a.v_cache = vc.p; a.q_out = in_place ? q.p : qo.p;
    a.page_table = table; a.row_start = row_start; a.kv_len = kv_len;
    a.q_norm = (const float *)qn.p; a.k_norm = (const float *)kn.p; a.rope = turned ? (const float *)rope.p : nullptr;
    a.ld_q = a.ld_k = a.ld_v = ld; a.ld_q_out = in_place ? ld : 0;
    a.in_dtype = in; a.dtype = out; a.batch = batch; a.rows = rows; a.heads = H; a.kv_heads = Hkv; a.head_dim = d;
    a.page_size = ps; a.num_pages = pages; a.max_pages = max_pages; a.qk_norm = mode; a.rope_len = rope_len; a.eps = 1e-6;
    if (qw_op_kv_append(&a, nullptr) != QW_OK) return fprintf(stderr, "%s\n", host_error.c_str()), 3;

    const Numbers &got_q = in_place ? q : qo;
    const int lo = in_place ? lq : wq;
    size_t wrong = 0;
    for (int r = 0; r < rows; r++)
        for (int i = 0; i < wq; i++) wrong += !(fabs(got_q[(size_t)r * lo + i] - want_q[(size_t)r * wq + i]) <= far_q[(size_t)r * wq + i]);
    for (size_t i = 0; i < cells; i++) wrong += !(fabs(kc[i] - want_k[i]) <= far_k[i]) || !(fabs(vc[i] - want_v[i]) <= far_v[i]);
    if (wrong) return fprintf(stderr, "%zu numbers are wrong\n", wrong), 1;
    return 0;
}
