/* Host-side rules on PhononCudaStatus words, plain C. */
#ifndef PHONON_STATUS_H
#define PHONON_STATUS_H

#include <stdint.h>

#include "phonon_cuda.h"

/* What a call that computes one stream's rows returns for the rows' status
 * words: a kernel that gave up a bounded wait says nothing about the values,
 * so its code goes before those of rows. */
static inline int phonon_rows_status(const int32_t *status, int rows) {
    int result = PHONON_CUDA_OK;
    for (int i = 0; i < rows; ++i) {
        if (status[i] == PHONON_CUDA_DEVICE_ERROR) return PHONON_CUDA_DEVICE_ERROR;
        if (status[i] != PHONON_CUDA_OK) result = PHONON_CUDA_NON_FINITE;
    }
    return result;
}

#endif
