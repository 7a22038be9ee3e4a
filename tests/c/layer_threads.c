/*
 * Two host threads that call the layer operators at once, without an
 * interpreter's lock between them. Built as a shared library by
 * tests/test_gpu_layers_limits.py, which owns the arrays.
 */
#include <pthread.h>
#include <stdatomic.h>

#include "geo/geo_b200.h"

typedef struct {
    const geo_b200_layer_norm_config_t *norm;
    const geo_b200_dropout_config_t *dropout;
    void *x, *weight, *bias, *y, *mean, *rstd, *y_bar, *z_bar, *residual_bar, *x_bar, *weight_bar, *bias_bar, *workspace;
    size_t workspace_bytes;
    cudaStream_t stream;
    int calls, refused;
} layer_loop_t;

static atomic_int waiting;

/* A layer norm, then its VJP behind residual and dropout, every other time with the cotangent of z. */
static void *run(void *argument) {
    layer_loop_t *a = argument;
    int i;
    atomic_fetch_sub(&waiting, 1);
    while (atomic_load(&waiting) > 0) {
    }
    for (i = 0; i < a->calls; ++i) {
        if (geo_b200_layer_norm(a->norm, a->x, a->weight, a->bias, a->y, a->mean, a->rstd, a->stream) != GEO_B200_OK)
            ++a->refused;
        if (geo_b200_residual_dropout_layer_norm_vjp(a->norm, a->dropout, NULL, a->x, a->weight, a->mean, a->rstd,
                                                     a->y_bar, i % 2 ? a->z_bar : NULL, a->residual_bar, a->x_bar,
                                                     a->weight_bar, a->bias_bar, a->workspace, a->workspace_bytes,
                                                     a->stream) != GEO_B200_OK)
            ++a->refused;
    }
    return NULL;
}

int layer_loops(layer_loop_t *first, layer_loop_t *second) {
    pthread_t threads[2];
    atomic_store(&waiting, 2);
    if (pthread_create(&threads[0], NULL, run, first) != 0) return 1;
    if (pthread_create(&threads[1], NULL, run, second) != 0) {
        atomic_store(&waiting, 0);
        pthread_join(threads[0], NULL);
        return 1;
    }
    pthread_join(threads[0], NULL);
    pthread_join(threads[1], NULL);
    return 0;
}
