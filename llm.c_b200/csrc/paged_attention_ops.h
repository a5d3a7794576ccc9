// What the two files of attention over pages share: the call, and which kernel takes it.
#pragma once
#include "paged.cuh"

struct PagedAttention {
    bf16* out;
    float* ws;
    const bf16* q;
    const long long* tree;
    long long ldo, ldq;
    int N, NH, layer;
    unsigned int* status;
};

// Tensor maps of a layer's keys and values, for copies of box_rows rows of a page by 64 channels of one head
int paged_maps(CUtensorMap* tmK, CUtensorMap* tmV, const PagedCache* c, int layer, int box_rows);

// A bound of the pieces of groups of `rows` query rows
inline long long paged_few_pieces(const PagedCache* c, int N, int NH, int rows) { return ((long long)N * (NH / c->heads) / rows + c->sequences) * c->heads; }
// Whether their units of keys fit 32-bit counts
bool paged_few_fits(const PagedCache* c, int N, int NH);

// Many rows to a cached head (paged_attention_wide.cu)
bool paged_wide(const PagedCache* c, int N, int NH);
long long paged_wide_workspace(const PagedCache* c, int N, int NH);
int paged_wide_launches(const PagedCache* c, int N, int NH);
int paged_wide_launch(const PagedCache* c, const PagedAttention& a, cudaStream_t stream);
