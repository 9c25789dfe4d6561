/*
 * Tests of the cache on pages in the nts:: host layer on a gfx950 GPU, beside nts_cache_tests: both types, with and without a causal
 * limit, sequences with a common beginning, what a call does besides its kernels, and tensors without memory.
 *
 *   nts_cache_layer_tests               run everything on device 0, exit 0 if all passed
 *   nts_cache_layer_tests --abort NAME  provoke one fatal error (no GPU needed)
 */
#include "../../niutensor_amd/nts/Cache.h"

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include <vector>

using namespace nts;

/* in place of the runtime's: counts the fills that the layer issues */
static int fills = 0;
extern "C" hipError_t hipMemset(void * dst, int value, size_t bytes)
{
    fills++;
    return hipMemsetD8((hipDeviceptr_t)dst, (unsigned char)value, bytes);
}

static const int DEV = 0;
static const int SEQS = 3, PAGE = 16, WIDTH = 40, KV = 2, HEADS = 4, DH = 16, PREFIX = 512;

static unsigned state = 54321;
/* multiples of 2^-8 between -1 and 1: the same in half */
static float Random()
{
    state = state * 1664525u + 1013904223u;
    return (float)((int)(state >> 23) - 256) / 256.0F;
}

static uint16_t ToHalf(float x)                     /* of such a multiple, or NaN */
{
    if (x != x)
        return 0x7e00;
    int e;
    const float f = frexpf(fabsf(x), &e);
    const uint16_t sign = x < 0 ? 0x8000 : 0;
    return x == 0 ? 0 : sign | (uint16_t)((e + 14) << 10) | ((uint16_t)(f * 2048.0F) & 0x3ff);
}

static float FromHalf(uint16_t h)
{
    const int e = (h >> 10) & 31, m = h & 0x3ff;
    const float x = e == 31 ? (m ? NAN : INFINITY) : (e == 0 ? ldexpf((float)m, -24) : ldexpf((float)(m | 0x400), e - 25));
    return h & 0x8000 ? -x : x;
}

static XTensor * Upload(int order, const int * dims, TENSOR_DATA_TYPE type, const std::vector<float> & host)
{
    XTensor * t = NewTensorV2(order, dims, type, 1.0F, DEV);
    std::vector<uint16_t> half(host.size());
    std::vector<int> ints(host.size());
    for (size_t i = 0; i < host.size(); i++) {
        half[i] = type == X_FLOAT16 ? ToHalf(host[i]) : 0;
        ints[i] = type == X_INT ? (int)host[i] : 0;
    }
    t->SetData(type == X_FLOAT16 ? (const void *)half.data() : (type == X_INT ? (const void *)ints.data() : (const void *)host.data()), t->unitNum);
    return t;
}

static std::vector<float> Download(const XTensor & t)
{
    std::vector<float> x(t.unitNum);
    if (t.dataType == X_FLOAT16) {
        std::vector<uint16_t> half(t.unitNum);
        t.GetData(half.data());
        for (int i = 0; i < t.unitNum; i++)
            x[i] = FromHalf(half[i]);
    }
    else
        t.GetData(x.data());
    return x;
}

static XTensor * Rows(int rows, int cols, TENSOR_DATA_TYPE type, std::vector<float> & host)
{
    const int dims[2] = {rows, cols};
    host.resize((size_t)rows * cols);
    for (float & x : host)
        x = Random();
    return Upload(2, dims, type, host);
}

/* Rows `from` on of out are sequence i's `fresh` last positions of `length` */
static bool Check(const std::vector<float> & out, int from, int fresh, int length, const std::vector<std::vector<float> > & k,
                  const std::vector<std::vector<float> > & v, const std::vector<float> & q, double scale, bool causal, bool half, const char * what)
{
    const double u = ldexp(1.0, -24), h = ldexp(1.0, -11), least = ldexp(1.0, -25);
    for (int t = 0; t < fresh; t++)
        for (int head = 0; head < HEADS; head++) {
            const int n = causal ? length - fresh + t + 1 : length, kh = head / (HEADS / KV);
            const float * x = &q[((size_t)(from + t) * HEADS + head) * DH];
            std::vector<double> s(n);
            double most = 0.0, product = 0.0, sum = 0.0;
            for (int j = 0; j < n; j++) {
                double a = 0.0;
                for (int c = 0; c < DH; c++) {
                    s[j] += (double)x[c] * k[j][kh * DH + c] * scale;
                    a += fabs((double)x[c] * k[j][kh * DH + c] * scale);
                }
                most = fmax(most, fabs(s[j]));
                product = fmax(product, a);
            }
            for (int j = 0; j < n; j++)
                sum += exp(s[j]);
            for (int c = 0; c < DH; c++) {
                double o = 0.0, a = 0.0, all = 0.0;
                for (int j = 0; j < n; j++) {
                    const double y = v[j][kh * DH + c];
                    o += exp(s[j]) / sum * y;
                    a += exp(s[j]) / sum * fabs(y);
                    all += fabs(y);
                }
                /* scores off by (dh + 2) 2^-24 of their products, probabilities and their sum by twice that each; exponentials, sums and
                   shifts by n + 64 + 4 |s| of 2^-24. Half: probabilities by 2^-11 or 2^-25, their sum if it is the rounded ones',
                   and the result */
                double tol = (4 * (DH + 2) * u * product + (n + 64 + 4 * most) * u) * a;
                if (half)
                    tol = (tol + h * a + least * all + fmax(h * fabs(o), least) + (h + least * n) * fabs(o)) * (1 + ldexp(1.0, -10));
                const double got = out[((size_t)(from + t) * HEADS + head) * DH + c];
                if (!(fabs(got - o) <= tol)) {
                    printf("%s: row %d head %d column %d: %g, expected %g within %g\n", what, from + t, head, c, got, o, tol);
                    return false;
                }
            }
        }
    return true;
}

static bool TestType(TENSOR_DATA_TYPE type)
{
    const bool half = type == X_FLOAT16;
    const int lengths[SEQS] = {600, 513, 561};
    /* the prefix on 32 pages of everyone, then each sequence's own */
    std::vector<float> table(SEQS * WIDTH), lens(lengths, lengths + SEQS);
    int pages = PREFIX / PAGE;
    for (int i = 0; i < SEQS; i++)
        for (int p = 0; p < WIDTH; p++)
            table[i * WIDTH + p] = p < PREFIX / PAGE ? PREFIX / PAGE - 1 - p : pages++;
    const size_t row = (size_t)KV * DH;
    std::vector<float> kPool((size_t)pages * PAGE * row, NAN), vPool(kPool);
    std::vector<std::vector<float> > k[SEQS], v[SEQS];
    std::vector<float> kNew, vNew, q;
    XTensor * kt = Rows(SEQS, KV * DH, type, kNew), * vt = Rows(SEQS, KV * DH, type, vNew), * qt = Rows(SEQS, HEADS * DH, type, q);
    for (int i = 0; i < SEQS; i++)
        for (int p = 0; p < lengths[i]; p++) {
            const size_t at = ((size_t)table[i * WIDTH + p / PAGE] * PAGE + p % PAGE) * row;
            const bool last = p == lengths[i] - 1;              /* comes by the call */
            for (size_t c = 0; c < row && !last && (i == 0 || p >= PREFIX); c++) {
                kPool[at + c] = Random();
                vPool[at + c] = Random();
            }
            k[i].push_back(last ? std::vector<float>(&kNew[i * row], &kNew[i * row] + row) : std::vector<float>(&kPool[at], &kPool[at] + row));
            v[i].push_back(last ? std::vector<float>(&vNew[i * row], &vNew[i * row] + row) : std::vector<float>(&vPool[at], &vPool[at] + row));
        }
    const int pool[4] = {pages, PAGE, KV, DH}, td[2] = {SEQS, WIDTH}, ld[1] = {SEQS};
    XTensor * keys = Upload(4, pool, type, kPool), * values = Upload(4, pool, type, vPool);
    XTensor * tt = Upload(2, td, X_INT, table), * lt = Upload(1, ld, X_INT, lens);
    AmdCacheBatch batch = {lt, NULL, tt, 1, 600};
    _AmdCacheAppend(keys, values, batch, kt, vt);

    bool ok = true;
    fills = 0;
    XTensor each = AmdAttentionCached(*keys, *values, batch, *qt, 0.25F);
    if (fills != 0) {
        printf("a step whose rows are all written fills its result %d times\n", fills);
        ok = false;
    }
    XTensor shared(&each);
    _AmdAttentionPrefix(keys, values, batch, qt, &shared, 0.25F, PREFIX);
    for (int i = 0; i < SEQS; i++) {
        ok = ok && Check(Download(each), i, 1, lengths[i], k[i], v[i], q, 0.25, true, half, "step");
        ok = ok && Check(Download(shared), i, 1, lengths[i], k[i], v[i], q, 0.25, true, half, "behind a prefix");
    }

    /* 3, 0 and 20 rows against all positions, one row of nobody behind them */
    std::vector<float> starts = {0, 3, 3, 23}, qMany;
    const int sd[1] = {SEQS + 1};
    XTensor * st = Upload(1, sd, X_INT, starts), * qm = Rows(24, HEADS * DH, type, qMany);
    AmdCacheBatch many = {lt, st, tt, 20, 0};
    XTensor all = AmdAttentionCached(*keys, *values, many, *qm, 0.25F, false), upTo = AmdAttentionCached(*keys, *values, many, *qm, 0.25F);
    for (int i = 0; i < SEQS; i++) {
        const int from = (int)starts[i], fresh = (int)starts[i + 1] - from;
        ok = ok && Check(Download(all), from, fresh, lengths[i], k[i], v[i], qMany, 0.25, false, half, "not causal");
        ok = ok && Check(Download(upTo), from, fresh, lengths[i], k[i], v[i], qMany, 0.25, true, half, "several rows");
    }
    /* rows of nobody: behind the starts, and behind a step of one row for every sequence */
    XTensor step = AmdAttentionCached(*keys, *values, batch, *qm, 0.25F);
    const std::vector<float> a = Download(all), b = Download(step);
    for (size_t c = 0; c < HEADS * DH; c++)
        ok = ok && a[23 * HEADS * DH + c] == 0 && b[3 * HEADS * DH + c] == 0 && b[23 * HEADS * DH + c] == 0;
    delete kt; delete vt; delete qt; delete keys; delete values; delete tt; delete lt; delete st; delete qm;
    return ok;
}

/* Tensors with shapes, some of them with made-up addresses: refused before any memory is looked at */
static XTensor * Shape(int order, int a, int b, int c, int d, TENSOR_DATA_TYPE type, bool data)
{
    const int dims[4] = {-a, b, c, d};
    XTensor * t = new XTensor(order, dims, type, 1.0F, 0, NULL);
    if (data)
        t->data = (void *)(uintptr_t)0x10000;
    return t;
}

static int Provoke(const char * name)
{
    XTensor * keys = Shape(4, 4, 8, 2, 16, X_FLOAT, true), * values = Shape(4, 4, 8, 2, 16, X_FLOAT, true);
    XTensor * lengths = Shape(1, 3, 0, 0, 0, X_INT, true), * pages = Shape(2, 3, 4, 0, 0, X_INT, true);
    XTensor * k = Shape(2, 3, 32, 0, 0, X_FLOAT, true), * q = Shape(2, 3, 64, 0, 0, X_FLOAT, true);
    AmdCacheBatch batch = {lengths, NULL, pages, 1, 0};
    if (!strcmp(name, "starts")) {
        batch.starts = Shape(1, 4, 0, 0, 0, X_INT, false);
        _AmdAttentionCached(keys, values, batch, q, q, 1.0F);
    }
    if (!strcmp(name, "rotation"))
        _AmdCacheAppend(keys, values, batch, k, k, Shape(3, 32, 8, 2, 0, X_FLOAT, false));
    if (!strcmp(name, "queries")) {
        XTensor * none = Shape(2, 3, 64, 0, 0, X_FLOAT, false);
        _AmdCacheAppend(keys, values, batch, k, k, NULL, false, none, none);
    }
    return 0;
}

int main(int argc, char ** argv)
{
    if (argc == 3 && !strcmp(argv[1], "--abort"))
        return Provoke(argv[2]);
    bool ok = true;
    const TENSOR_DATA_TYPE types[2] = {X_FLOAT, X_FLOAT16};
    for (int i = 0; i < 2; i++) {
        const bool passed = TestType(types[i]);
        printf(">> %-36s %s\n", i == 0 ? "TestCacheLayer, float" : "TestCacheLayer, half", passed ? "passed" : "FAILED");
        ok = ok && passed;
    }
    printf(ok ? "OK! Everything is good!\n" : "Sorry, some problems happened!\n");
    return ok ? 0 : 1;
}
