// The products of a Newton-Schulz step on a batch of matrices (muon_gemm.hip), and the matrices of a batch.
#pragma once

#include "values.h"

namespace wf {

constexpr int kMuonBatch = 128;             // matrices a launch: their addresses are kernel arguments

// What is stepped, matrix by matrix: p (of type dt) becomes keep p - rate O, O the orthogonalised update.
struct MuonTensors {
    void* p[kMuonBatch];
    const void* g[kMuonBatch];
    float* m[kMuonBatch];                  // NULL: the update is g itself
    int dt;
    float keep, rate;                      // keep 0: p is written only
    float mu, nu;                          // m = mu m + nu g, nu = 1 - mu; the update is mu m + nu g (nesterov), or m
    int nesterov;
};

// A batch in float16, matrix b at x + b (rows ld), X s with s a power of two; symmetric matrices [side, sld], times s^2; rows' lengths ld, sld are
// multiples of 8, zeros past the matrix.
struct MuonShape {
    int rows, cols, ld, side, sld, batch;
    bool tall;                             // rows > cols: the short side is the columns
};

// out = alpha S + beta in + gamma I, S = x x^T (or x^T x where tall), in may be NULL
struct MuonSymmetric {
    const uint16_t* x;                     // [rows, ld], or a symmetric matrix [side, sld] (square set)
    bool square;
    const uint16_t* in;
    uint16_t* out;
    float alpha, beta, gamma;
};
// next = alpha q x (x q where tall) + a (x + lo / 2048); the remainder of its rounding, times 2048, to lo. lo NULL: next = alpha q x
// alone; next NULL: the tensors' step with it.
struct MuonUpdate {
    const uint16_t *x, *q;
    uint16_t *lo, *next;
    float alpha, a;
};

// how a batch's products run: the tiling of a symmetric product (square: of A, else of X) and its slices of the sum, of the update
void muon_symmetric_form(const MuonShape& s, bool square, int& tiling, int& slices);
int muon_update_tiling(const MuonShape& s);

int64_t muon_symmetric_bytes(const MuonShape& s, bool square);      // of float32 partial sums
void muon_symmetric(const MuonShape& s, const MuonSymmetric& q, float* parts, hipStream_t st);
void muon_update(const MuonShape& s, const MuonUpdate& q, const MuonTensors& t, hipStream_t st);

}  // namespace wf
