/*
 * gguf_hip_packed.h — calls of entry points by number, their arguments as one array: for
 * hosts whose foreign calls cost by the argument.
 */
#ifndef GGUF_HIP_PACKED_H
#define GGUF_HIP_PACKED_H

#include "gguf_hip_paged.h"
#include "gguf_hip_sample.h"

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

#define GGUF_HIP_PACKED_PAGED_APPEND 0
#define GGUF_HIP_PACKED_PAGED_ATTENTION 1
#define GGUF_HIP_PACKED_PAGED_LOAD 2
#define GGUF_HIP_PACKED_PAGED_FORK 3
#define GGUF_HIP_PACKED_PAGED_GROW 4
#define GGUF_HIP_PACKED_PAGED_COMPACT 5
#define GGUF_HIP_PACKED_SAMPLE 6

/* Entry point `op` with the arguments of its declaration in order, eight bytes each: a
 * pointer, an integer as int64_t (one that its parameter cannot hold is refused), a float in
 * the first four.  `bytes` has to be eight times their number.  Returns what it returns. */
int gguf_hip_packed_call(int op, const void *args, int64_t bytes);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif

#endif /* GGUF_HIP_PACKED_H */
