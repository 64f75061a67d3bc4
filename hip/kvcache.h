/*
 * nvshare-amd: arguments of the paged key/value cache's kernels
 * (libnvshare_hiputil.so).  Strides are in values, not bytes.
 */
#ifndef NVS_KVCACHE_H
#define NVS_KVCACHE_H

#include <stdint.h>

enum { NVS_KV_BF16 = 0, NVS_KV_FP16 = 1, NVS_KV_E4M3 = 2 };

/* The cache and the step's sequences. */
struct nvs_kv {
	void *k_cache, *v_cache;
	const float *k_scale, *v_scale; /* [kv_heads], e4m3 only */
	const int *table;		/* [batch][per_seq] pages */
	const int *lens;		/* [batch], the new tokens included */
	const int *starts;		/* [batch + 1] rows, or null */
	int64_t table_row;
	int64_t k_page, k_slot, k_head;
	int64_t v_page, v_slot, v_head;
	int type, cache_type;
	int batch, total;		/* sequences, rows */
	int heads, kv_heads, dim;
	int pages, page_size, per_seq;
};

struct nvs_kv_append_args {
	const void *q, *k, *v; /* q may be null */
	void *q_out;
	const float *rotation; /* [positions][cosines, sines], or null */
	int64_t q_row, q_head, k_row, k_head, v_row, v_head;
	int64_t q_out_row, q_out_head, rotation_row;
	int rotary, interleaved;
	int fill; /* rows of no sequence: zeros, or left as they were */
};

struct nvs_kv_attend_args {
	const void *q;
	void *out;
	float *lse; /* [total][heads], or null */
	int64_t q_row, q_head, out_row, out_head;
	float scale;
	int window;  /* keys that a query sees, itself included; 0: all */
	int max_new; /* no sequence has more rows than this */
	int fill;
};

#endif
