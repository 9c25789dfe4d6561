/*
 * Tests of the cache on pages in the nts:: host layer on a gfx950 GPU: prompts enter, a step of one token each follows, the
 * sequences attend to what stands in the pools, and all of it is compared with the formulas in double on the host.
 *
 *   nts_cache_tests               run everything on device 0, exit 0 if all passed
 *   nts_cache_tests --abort NAME  provoke one fatal error (no GPU needed)
 */
#include "../../niutensor_amd/nts/Cache.h"

#include <math.h>
#include <stdio.h>
#include <string.h>
#include <vector>

using namespace nts;

static const int DEV = 0;
static const int SEQS = 3, PAGE = 4, WIDTH = 5, PAGES = 16, KV = 2, HEADS = 4, DH = 8, ROT = 6, POS = WIDTH * PAGE;

static unsigned state = 12345;
static float Random()
{
    state = state * 1664525u + 1013904223u;
    return (float)(state >> 8) / (1 << 23) - 1.0F;
}

static XTensor * Floats(int rows, int cols, std::vector<float> & host)
{
    int dims[2] = {rows, cols};
    host.resize((size_t)rows * cols);
    for (float & x : host)
        x = Random();
    XTensor * t = NewTensorV2(2, dims, X_FLOAT, 1.0F, DEV);
    t->SetData(host.data(), t->unitNum);
    return t;
}

static XTensor * Ints(int rows, int cols, const std::vector<int> & host)
{
    int dims[2] = {rows, cols};
    XTensor * t = cols > 0 ? NewTensorV2(2, dims, X_INT, 1.0F, DEV) : NewTensorV2(1, dims, X_INT, 1.0F, DEV);
    t->SetData(host.data(), t->unitNum);
    return t;
}

/* columns j and j + ROT / 2 of every head, turned by the angle of position p */
static void Turn(double * head, int p)
{
    for (int j = 0; j < ROT / 2; j++) {
        const double c = (float)cos(p * pow(100.0, -2.0 * j / ROT)), s = (float)sin(p * pow(100.0, -2.0 * j / ROT));
        const double x = head[j], y = head[j + ROT / 2];
        head[j] = x * c - y * s;
        head[j + ROT / 2] = y * c + x * s;
    }
}

/* the turned keys and the values of the sequences, in the order of their positions, and the new tokens' results */
struct Reference {
    std::vector<std::vector<double> > k[SEQS], v[SEQS];

    bool Step(const std::vector<int> & starts, const std::vector<float> & k0, const std::vector<float> & v0,
              const std::vector<float> & q0, const std::vector<float> & got, double scale, const char * what)
    {
        for (int i = 0; i < SEQS; i++) {
            const size_t before = k[i].size();
            for (int t = starts[i]; t < starts[i + 1]; t++) {
                std::vector<double> a(k0.begin() + t * KV * DH, k0.begin() + (t + 1) * KV * DH);
                for (int h = 0; h < KV; h++)
                    Turn(&a[h * DH], (int)k[i].size());
                k[i].push_back(a);
                v[i].push_back(std::vector<double>(v0.begin() + t * KV * DH, v0.begin() + (t + 1) * KV * DH));
            }
            for (int t = starts[i]; t < starts[i + 1]; t++)
                for (int h = 0; h < HEADS; h++) {
                    const int own = (int)before + t - starts[i], kh = h / (HEADS / KV);
                    std::vector<double> q(q0.begin() + (t * HEADS + h) * DH, q0.begin() + (t * HEADS + h + 1) * DH);
                    Turn(q.data(), own);
                    std::vector<double> out(DH, 0.0);
                    double sum = 0.0;
                    for (int j = 0; j <= own; j++) {
                        double s = 0.0;
                        for (int c = 0; c < DH; c++)
                            s += q[c] * k[i][j][kh * DH + c];
                        const double e = exp(s * scale);
                        sum += e;
                        for (int c = 0; c < DH; c++)
                            out[c] += e * v[i][j][kh * DH + c];
                    }
                    for (int c = 0; c < DH; c++) {
                        /* in units of 2^-24, with values below 1 and turned columns below 1.5, so that scale sum |q k| is below 9: a score is
                           off by 10 * 9 for its product and 4 * 9 for the turns of q and k, the quotient by four times that; sums,
                           exponentials and shifts of 15 keys by 15 + 64 + 4 * 9 */
                        const double x = got[(t * HEADS + h) * DH + c];
                        if (!(fabs(x - out[c] / sum) <= (4 * 126 + 115) / 16777216.0)) {
                            printf("%s: token %d head %d column %d: %g, expected %g\n", what, t, h, c, x, out[c] / sum);
                            return false;
                        }
                    }
                }
        }
        return true;
    }
};

static bool TestCache()
{
    int pool[4] = {PAGES, PAGE, KV, DH}, rot[3] = {POS, ROT / 2, 2};
    std::vector<float> nans((size_t)PAGES * PAGE * KV * DH, NAN), table;
    XTensor * keys = NewTensorV2(4, pool, X_FLOAT, 1.0F, DEV);
    XTensor * values = NewTensorV2(4, pool, X_FLOAT, 1.0F, DEV);
    keys->SetData(nans.data(), keys->unitNum);
    values->SetData(nans.data(), values->unitNum);
    for (int p = 0; p < POS; p++)
        for (int j = 0; j < ROT / 2; j++) {
            table.push_back((float)cos(p * pow(100.0, -2.0 * j / ROT)));
            table.push_back((float)sin(p * pow(100.0, -2.0 * j / ROT)));
        }
    XTensor * rotation = NewTensorV2(3, rot, X_FLOAT, 1.0F, DEV);
    rotation->SetData(table.data(), rotation->unitNum);
    std::vector<int> pages;
    for (int i = 0; i < SEQS * WIDTH; i++)
        pages.push_back((7 * i + 3) % PAGES);
    XTensor * pageTable = Ints(SEQS, WIDTH, pages);

    Reference ref;
    bool ok = true;
    /* prompts of 5, 1 and 9 tokens, then twice one token each */
    std::vector<int> starts = {0, 5, 6, 15}, lengths = {5, 1, 9};
    for (int step = 0; step < 3 && ok; step++) {
        if (step > 0) {
            starts = {0, 1, 2, 3};
            for (int & x : lengths)
                x++;
        }
        const int tokens = starts[SEQS];
        std::vector<float> k0, v0, q0, got;
        XTensor * k = Floats(tokens, KV * DH, k0), * v = Floats(tokens, KV * DH, v0), * q = Floats(tokens, HEADS * DH, q0);
        XTensor * l = Ints(SEQS, 0, lengths), * s = Ints(SEQS + 1, 0, starts);
        AmdCacheBatch batch = {l, step == 0 ? s : NULL, pageTable, step == 0 ? 9 : 1, 0};
        _AmdCacheAppend(keys, values, batch, k, v, rotation, false, q, q);
        XTensor out = AmdAttentionCached(*keys, *values, batch, *q, 0.5F);
        got.resize(out.unitNum);
        out.GetData(got.data());
        ok = ref.Step(starts, k0, v0, q0, got, 0.5, "attention");
        /* nothing in common is a prefix too */
        XTensor again(&out);
        _AmdAttentionPrefix(keys, values, batch, q, &again, 0.5F, 0);
        std::vector<float> same(again.unitNum);
        again.GetData(same.data());
        ok = ok && memcmp(same.data(), got.data(), got.size() * sizeof(float)) == 0;
        delete k; delete v; delete q; delete l; delete s;
    }
    delete keys; delete values; delete rotation; delete pageTable;
    return ok;
}

/* Calls that are refused before any memory is looked at: tensors with shapes and made-up addresses */
static XTensor * Shape(int order, int a, int b, int c, int d, TENSOR_DATA_TYPE type)
{
    int dims[4] = {-a, b, c, d};
    XTensor * t = new XTensor(order, dims, type, 1.0F, 0, NULL);
    return t;
}

static int Provoke(const char * name)
{
    XTensor * keys = Shape(4, 4, 8, 2, 16, X_FLOAT), * values = Shape(4, 4, 8, 2, 16, X_FLOAT);
    XTensor * half = Shape(2, 3, 64, 0, 0, X_FLOAT16), * q = Shape(2, 3, 64, 0, 0, X_FLOAT), * odd = Shape(2, 3, 60, 0, 0, X_FLOAT);
    XTensor * k = Shape(2, 3, 32, 0, 0, X_FLOAT), * lengths = Shape(1, 3, 0, 0, 0, X_INT), * pages = Shape(2, 3, 4, 0, 0, X_INT);
    XTensor * floats = Shape(1, 3, 0, 0, 0, X_FLOAT);
    AmdCacheBatch batch = {lengths, NULL, pages, 1, 0};
    if (!strcmp(name, "type"))
        _AmdAttentionCached(keys, values, batch, half, half, 1.0F);
    if (!strcmp(name, "hidden"))
        _AmdAttentionCached(keys, values, batch, odd, odd, 1.0F);
    if (!strcmp(name, "shape"))
        _AmdCacheAppend(keys, values, batch, q, q);
    if (!strcmp(name, "empty"))
        _AmdCacheAppend(keys, values, batch, k, k, NULL, false, q, NULL);
    if (!strcmp(name, "starts")) {
        batch.starts = lengths;
        _AmdAttentionCached(keys, values, batch, q, q, 1.0F);
    }
    if (!strcmp(name, "integers")) {
        batch.lengths = floats;
        _AmdAttentionCached(keys, values, batch, q, q, 1.0F);
    }
    if (!strcmp(name, "prefix"))
        _AmdAttentionPrefix(keys, values, batch, q, q, 1.0F, -1);
    if (!strcmp(name, "abi"))                           /* shapes without memory: refused below this layer */
        _AmdAttentionCached(keys, values, batch, q, q, 1.0F);
    return 0;
}

int main(int argc, char ** argv)
{
    if (argc == 3 && !strcmp(argv[1], "--abort"))
        return Provoke(argv[2]);
    const bool ok = TestCache();
    printf(">> %-36s %s\n", "TestCache", ok ? "passed" : "FAILED");
    printf(ok ? "OK! Everything is good!\n" : "Sorry, some problems happened!\n");
    return ok ? 0 : 1;
}
