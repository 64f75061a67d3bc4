/*
 * nvshare-amd: the calls of nvshare_amd.kvcache (_kvbind.so).
 *
 * A step of a few tokens takes the GPU a few microseconds, and looking its
 * dozen tensors over in Python three times as long: so arguments are
 * checked, results allocated and kernels launched here.  Every check of
 * the Python module's documentation is in this file, for tensors on the
 * CPU too; only what it names is launched, on the stream that it is given.
 */
#include <ATen/MemoryOverlap.h>
#include <torch/extension.h>

#include <dlfcn.h>

#include <cmath>
#include <limits>
#include <optional>
#include <sstream>

#include "kvcache.h"

namespace {

using at::Tensor;
using Maybe = std::optional<Tensor>;

/* The kernels' library, which lies beside this one.  It is loaded for the
 * first launch only: tensors on the CPU need neither it nor a GPU's runtime.
 */
struct entries {
	int (*append)(const nvs_kv *c, const nvs_kv_append_args *a,
		      void *stream);
	int64_t (*attend_work)(const nvs_kv *c, const nvs_kv_attend_args *a);
	int (*attend)(const nvs_kv *c, const nvs_kv_attend_args *a, void *work,
		      void *stream);
};

const entries &kernels()
{
	static const entries e = [] {
		void *lib = dlopen("libnvshare_hiputil.so",
				   RTLD_NOW | RTLD_LOCAL);
		auto entry = [&](const char *name) {
			void *p = lib ? dlsym(lib, name) : nullptr;

			if (!p)
				throw std::runtime_error(
					std::string(dlerror()) +
					"; build with `make -C hip` (hipcc, "
					"gfx950)");
			return p;
		};
		entries got;

		got.append = (decltype(got.append))entry("nvs_kv_append");
		got.attend_work = (decltype(got.attend_work))entry(
			"nvs_kv_attend_work");
		got.attend = (decltype(got.attend))entry("nvs_kv_attend");
		return got;
	}();
	return e;
}

constexpr int64_t MOST = std::numeric_limits<int32_t>::max();

template <typename... Args> [[noreturn]] void refuse(const Args &...args)
{
	std::ostringstream s;

	(s << ... << args);
	throw pybind11::value_error(s.str());
}

std::string shown(const Tensor &t)
{
	std::ostringstream s;

	s << t.scalar_type() << " " << t.sizes() << " on " << t.device();
	return s.str();
}

/* Rows of heads: [total, heads, dim]. */
void check_rows(const char *name, const Tensor &t)
{
	if (t.dim() != 3)
		refuse(name, ": [total, heads, dim] is wanted, got ", shown(t));
	if (t.scalar_type() != at::kBFloat16 && t.scalar_type() != at::kHalf)
		refuse(name, ": bfloat16 or float16 is wanted, got ", shown(t));
	if (t.size(0) * t.size(1) >= MOST)
		refuse(name, ": ", t.size(0), " rows of ", t.size(1),
		       " heads pass 31 bits");
}

/* `t` has the rows, type and device of `k`, and its heads or others. */
void check_like(const char *name, const Tensor &t, const Tensor &k,
		bool heads)
{
	if (t.dim() != 3 || t.scalar_type() != k.scalar_type() ||
	    t.device() != k.device() || t.size(0) != k.size(0) ||
	    t.size(2) != k.size(2) || (!heads && t.size(1) != k.size(1)))
		refuse(name, ": ", shown(t), " does not go with ", shown(k));
}

/* Each head's values are contiguous and begin at 16 bytes. */
void check_strides(const char *name, const Tensor &t, int64_t step)
{
	bool fine = t.stride(-1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0;

	for (int64_t d = 0; d + 1 < t.dim(); d++)
		fine &= t.size(d) == 1 || t.stride(d) % step == 0;
	if (!fine)
		refuse(name, ": values of a head are not contiguous at 16 bytes"
			     " (strides ",
		       t.strides(), ")");
}

/* A stride that is never taken is none. */
int64_t step(const Tensor &t, int64_t d)
{
	return t.size(d) == 1 ? 0 : t.stride(d);
}

/* Nothing in `t`, which is written, is in two places. */
void check_distinct(const char *name, const Tensor &t)
{
	for (int64_t d = 0; d < t.dim(); d++)
		if (t.size(d) > 1 && t.stride(d) == 0)
			refuse(name, ": an expanded tensor cannot be written "
				     "to (strides ",
			       t.strides(), ")");
}

/* Nor is it in a place of `other`, as far as torch can tell cheaply: blocks
 * read and write in any order. */
void check_apart(const char *name, const Tensor &t, const Tensor &other,
		 bool same_allowed = false)
{
	const at::MemOverlapStatus status = at::get_overlap_status(t, other);

	if (status == at::MemOverlapStatus::Partial ||
	    (status == at::MemOverlapStatus::Full && !same_allowed))
		refuse(name, ": shares memory with other arguments");
}

void check_index(const char *name, const Tensor &t, int64_t n,
		 const Tensor &rows)
{
	if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n ||
	    t.device() != rows.device() || !t.is_contiguous())
		refuse(name, ": a contiguous int32 [", n,
		       "] tensor on the rows' device is wanted, got ",
		       shown(t));
}

void check_scale(const char *name, const Maybe &s, const Tensor &cache)
{
	const bool e4m3 = cache.scalar_type() == at::kFloat8_e4m3fn;

	if (s.has_value() != e4m3)
		refuse(name, ": wanted with float8_e4m3fn, and only there");
	if (e4m3 && (s->scalar_type() != at::kFloat || s->dim() != 1 ||
		     s->size(0) != cache.size(2) ||
		     s->device() != cache.device() || !s->is_contiguous()))
		refuse(name, ": a contiguous float32 [", cache.size(2),
		       "] tensor on the cache's device is wanted, got ",
		       shown(*s));
}

void *at_of(const Maybe &t)
{
	return t ? t->data_ptr() : nullptr;
}

/* What both operators ask of their common arguments. */
nvs_kv describe(const Tensor &ck, const Tensor &cv, const Maybe &k_scale,
		const Maybe &v_scale, const Tensor &rows, int64_t heads,
		const Tensor &table, const Tensor &lens, const Maybe &starts)
{
	const int64_t total = rows.size(0), dim = rows.size(2);

	if (ck.dim() != 4 || ck.sizes() != cv.sizes() ||
	    ck.scalar_type() != cv.scalar_type() || ck.size(3) != dim ||
	    ck.device() != rows.device() || cv.device() != rows.device())
		refuse("cache: keys ", shown(ck), " and values ", shown(cv),
		       " are not both [pages, page_size, kv_heads, ", dim,
		       "] on ", rows.device());
	const int64_t pages = ck.size(0), page_size = ck.size(1);
	const int64_t kv_heads = ck.size(2);

	if (heads == 0 || kv_heads == 0 || heads % kv_heads || pages == 0 ||
	    page_size == 0 || pages > MOST || page_size > MOST)
		refuse("cache: ", pages, " pages of ", page_size, " with ",
		       kv_heads, " heads cannot serve ", heads, " heads");
	const bool e4m3 = ck.scalar_type() == at::kFloat8_e4m3fn;

	if (!e4m3 && ck.scalar_type() != rows.scalar_type())
		refuse("cache: ", ck.scalar_type(), " is neither ",
		       rows.scalar_type(), " nor float8_e4m3fn");
	check_scale("k_scale", k_scale, ck);
	check_scale("v_scale", v_scale, ck);
	if (table.scalar_type() != at::kInt || table.dim() != 2 ||
	    table.device() != rows.device() ||
	    (table.size(1) > 1 && table.stride(1) != 1))
		refuse("table: an int32 [batch, pages] tensor with contiguous "
		       "rows on the rows' device is wanted, got ",
		       shown(table));
	const int64_t batch = table.size(0), per_seq = table.size(1);

	if (batch >= MOST || per_seq * page_size > MOST)
		refuse("table: ", batch, " sequences, or ", per_seq,
		       " pages of ", page_size, ", pass 31 bits");
	check_index("lens", lens, batch, rows);
	if (starts)
		check_index("starts", *starts, batch + 1, rows);
	else if (batch ? total % batch : total)
		refuse(total, " rows are not the same number for each of ",
		       batch, " sequences: give starts");
	if (total && (batch == 0 || per_seq == 0))
		refuse("table: rows, but no sequences or no pages");
	if (rows.is_cuda()) {
		check_strides("cache.k", ck, e4m3 ? 16 : 8);
		check_strides("cache.v", cv, e4m3 ? 16 : 8);
	}

	const int type = rows.scalar_type() == at::kHalf ? NVS_KV_FP16 :
							   NVS_KV_BF16;
	nvs_kv c = {};

	c.k_cache = ck.data_ptr();
	c.v_cache = cv.data_ptr();
	c.k_scale = (const float *)at_of(k_scale);
	c.v_scale = (const float *)at_of(v_scale);
	c.table = (const int *)table.data_ptr();
	c.lens = (const int *)lens.data_ptr();
	c.starts = (const int *)at_of(starts);
	c.table_row = step(table, 0);
	c.k_page = step(ck, 0);
	c.k_slot = step(ck, 1);
	c.k_head = step(ck, 2);
	c.v_page = step(cv, 0);
	c.v_slot = step(cv, 1);
	c.v_head = step(cv, 2);
	c.type = type;
	c.cache_type = e4m3 ? NVS_KV_E4M3 : type;
	c.batch = (int)batch;
	c.total = (int)total;
	c.heads = (int)heads;
	c.kv_heads = (int)kv_heads;
	c.dim = (int)dim;
	c.pages = (int)pages;
	c.page_size = (int)page_size;
	c.per_seq = (int)per_seq;
	return c;
}

/* Whether a derivative is wanted of a call with `t`: backwards, or
 * forwards (a dual tensor, a transform's), which no_grad leaves on. */
bool differentiated(const Tensor &t)
{
	if (at::GradMode::is_enabled() && t.requires_grad())
		return true;
	return c10::AutogradState::get_tls_state().get_fw_grad_mode() &&
	       t._fw_grad(0).defined();
}

void forward_only(std::initializer_list<const Tensor *> tensors,
		  std::initializer_list<const Maybe *> optional)
{
	bool wanted = false;

	for (const Tensor *t : tensors)
		wanted |= differentiated(*t);
	for (const Maybe *t : optional)
		wanted |= *t && differentiated(**t);
	if (wanted)
		refuse("forward only: detach the arguments, or, where none "
		       "is a dual tensor, call under torch.no_grad()");
}

/* A kernel writes to `t`: autograd has to see that what it may have saved
 * of it is gone.  (Tensors on the CPU are written to by torch.) */
void written(const Tensor &t)
{
	if (!t.is_inference())
		t.unsafeGetTensorImpl()->bump_version();
}

void launched(const char *what, int error)
{
	if (error)
		throw std::runtime_error(std::string(what) +
					 " failed with hipError_t=" +
					 std::to_string(error));
}

/* The rotated queries, if there are any; nothing is launched for tensors
 * on the CPU. */
Maybe append(const Tensor &ck, const Tensor &cv, const Maybe &k_scale,
	     const Maybe &v_scale, const Tensor &k, const Tensor &v,
	     const Tensor &table, const Tensor &lens, const Maybe &starts,
	     const Maybe &q, const Maybe &rotation, bool interleaved,
	     Maybe q_out, uintptr_t stream)
{
	check_rows("k", k);
	check_like("v", v, k, false);
	if (q) {
		check_rows("q", *q);
		check_like("q", *q, k, true);
	} else if (q_out)
		refuse("q_out without q");
	const nvs_kv c = describe(ck, cv, k_scale, v_scale, k,
				  q ? q->size(1) : k.size(1), table, lens,
				  starts);

	if (k.size(1) != c.kv_heads)
		refuse("k: ", shown(k), " does not go with the cache's ",
		       c.kv_heads, " heads");
	if (c.dim == 0 || c.dim % 16)
		refuse("dim ", c.dim, " is no multiple of 16");
	nvs_kv_append_args a = {};

	if (rotation) {
		if (rotation->dim() != 2 ||
		    rotation->scalar_type() != at::kFloat ||
		    rotation->device() != k.device())
			refuse("rotation: a float32 [positions, rotary] tensor "
			       "on the device of k is wanted, got ",
			       shown(*rotation));
		const int64_t rotary = rotation->size(1);

		if (rotary == 0 || rotary % 16 || rotary > c.dim)
			refuse("rotation: ", rotary,
			       " dimensions are no multiple of 16 up to ",
			       c.dim);
		if (rotation->size(0) < (int64_t)c.per_seq * c.page_size)
			refuse("rotation: ", rotation->size(0),
			       " positions, the table names ",
			       (int64_t)c.per_seq * c.page_size);
		a.rotation = (const float *)rotation->data_ptr();
		a.rotation_row = step(*rotation, 0);
		a.rotary = (int)rotary;
		a.interleaved = interleaved;
	}
	forward_only({ &ck, &cv, &k, &v },
		     { &k_scale, &v_scale, &q, &rotation, &q_out });
	check_distinct("cache", ck);
	check_distinct("cache", cv);
	check_apart("cache", ck, cv);
	for (const Tensor *t : { &k, &v }) {
		check_apart("cache", ck, *t);
		check_apart("cache", cv, *t);
	}
	a.fill = !q_out;
	if (q && !q_out)
		q_out = at::empty(q->sizes(), q->options());
	else if (q) {
		check_like("q_out", *q_out, *q, false);
		check_distinct("q_out", *q_out);
		check_apart("q_out", *q_out, *q, true);
		for (const Tensor *t : { &k, &v, &ck, &cv })
			check_apart("q_out", *q_out, *t);
	}
	if (c.total == 0 || !k.is_cuda())
		return q_out;
	check_strides("k", k, 8);
	check_strides("v", v, 8);
	if (q) {
		check_strides("q", *q, 8);
		check_strides("q_out", *q_out, 8);
		a.q = q->data_ptr();
		a.q_row = step(*q, 0);
		a.q_head = step(*q, 1);
		a.q_out = q_out->data_ptr();
		a.q_out_row = step(*q_out, 0);
		a.q_out_head = step(*q_out, 1);
	}
	if (rotation)
		check_strides("rotation", *rotation, 4);
	a.k = k.data_ptr();
	a.k_row = step(k, 0);
	a.k_head = step(k, 1);
	a.v = v.data_ptr();
	a.v_row = step(v, 0);
	a.v_head = step(v, 1);
	written(ck);
	written(cv);
	if (q)
		written(*q_out);
	launched("kv_append", kernels().append(&c, &a, (void *)stream));
	return q_out;
}

/* The result and its logarithms; as above for tensors on the CPU. */
std::pair<Tensor, Maybe> attend(const Tensor &ck, const Tensor &cv,
				const Maybe &k_scale, const Maybe &v_scale,
				const Tensor &q, const Tensor &table,
				const Tensor &lens, const Maybe &starts,
				std::optional<double> given_scale,
				int64_t window,
				std::optional<int64_t> max_new,
				Maybe out, bool want_lse, uintptr_t stream)
{
	check_rows("q", q);
	const nvs_kv c = describe(ck, cv, k_scale, v_scale, q, q.size(1),
				  table, lens, starts);

	if (c.dim != 64 && c.dim != 128 && c.dim != 256)
		refuse("dim ", c.dim, " is not one of 64, 128 and 256");
	forward_only({ &ck, &cv, &q }, { &k_scale, &v_scale, &out });
	const double scale = given_scale.value_or(std::pow(c.dim, -0.5));

	if (!std::isfinite((float)scale))
		refuse("scale ", scale, " is not finite in 32 bits");
	nvs_kv_attend_args a = {};

	a.fill = !out;
	if (!out)
		out = at::empty(q.sizes(), q.options());
	else {
		check_like("out", *out, q, false);
		check_distinct("out", *out);
		check_apart("out", *out, q, true);
		check_apart("out", *out, ck);
		check_apart("out", *out, cv);
	}
	Maybe lse;

	if (want_lse) {
		lse = at::empty({ q.size(0), q.size(1) },
				q.options().dtype(at::kFloat));
		a.lse = (float *)lse->data_ptr();
	}
	if (c.total == 0 || !q.is_cuda())
		return { *out, lse };
	check_strides("q", q, 8);
	check_strides("out", *out, 8);
	a.q = q.data_ptr();
	a.q_row = step(q, 0);
	a.q_head = step(q, 1);
	a.out = out->data_ptr();
	a.out_row = step(*out, 0);
	a.out_head = step(*out, 1);
	a.scale = (float)scale;
	a.window = (int)std::min(window, MOST);
	a.max_new = (int)std::min(max_new.value_or(q.size(0)), q.size(0));
	const int64_t bytes = kernels().attend_work(&c, &a);

	if (bytes < 0)
		launched("kv_attend", 1);
	Tensor work;

	if (bytes)
		work = at::empty({ bytes }, q.options().dtype(at::kByte));
	written(*out);
	launched("kv_attend",
		 kernels().attend(&c, &a, bytes ? work.data_ptr() : nullptr,
				  (void *)stream));
	return { *out, lse };
}

} /* namespace */

PYBIND11_MODULE(_kvbind, m)
{
	m.def("append", &append);
	m.def("attend", &attend);
}
