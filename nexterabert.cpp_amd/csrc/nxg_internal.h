// nxg_internal.h -- declarations shared by the host and device halves of libnxg.
#ifndef NXG_INTERNAL_H
#define NXG_INTERNAL_H

#include <stddef.h>
#include <stdint.h>

// Copies rows of n_in int8 values (row-major) into 16-row x 64-input fragment
// tiles: byte (r, k) goes to ((r/16)*KS + k/64)*1024 + ((r%16) + 16*((k%64)/16))*16 + k%16.
// `tiled` must be zero-filled and hold ceil(n_rows/16)*16 * KS*64 bytes. n_in % 16 == 0.
void nxg_tile_rows(const int8_t * rows, int n_rows, int n_in, int KS, int8_t * tiled);

// Records the message returned by nxg_last_error() on this thread.
void nxg_set_error(const char * msg);

// Records a formatted message and returns `code`.
int nxg_fail(int code, const char * fmt, ...) __attribute__((format(printf, 2, 3)));

// NXG_OK if the current device is a gfx950 GPU.
int nxg_check_device(void);

// Compute units of the current device (256 without a gfx950 GPU): the same on every thread, so that a workspace's size
// and the call that uses it have one plan.
int nxg_device_cus(void);

// NXG_OK, or NXG_EDEVICE with the error of the launch just made.
int nxg_launch_check(const char * what);

#endif
