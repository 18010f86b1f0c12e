"""CPU: what the biased attention and the group normalisation refuse, at the C ABI (before anything is launched) and in Python, and the layout of the
attention descriptor."""
import ctypes

import pytest
import torch

NULL, SHAPE, DTYPE, ALIGN, UNSUPPORTED, SCRATCH = -4, -1, -2, -3, -5, -6


def test_descriptor_layout_matches_header():
	import vit_amd._lib as L
	D = L.BiasedAttentionDesc
	# 10 pointers, 22 int64, table + lookup, 3 int64, 2 pointers, 2 int64, 4 pointers, prep + bytes, workspace + bytes, 2 floats, 3 int32 (+ 4 of padding)
	assert ctypes.sizeof(D) == 8 * (10 + 22 + 2 + 3 + 2 + 2 + 4 + 2 + 2) + 2 * 4 + 3 * 4 + 4
	assert D.B.offset == 80 and D.table.offset == 80 + 22 * 8 and D.scale.offset == ctypes.sizeof(D) - 24


def desc(**kw):
	import vit_amd._lib as L
	buf = ctypes.create_string_buffer(8192 + 256)
	p = (ctypes.addressof(buf) + 255) & ~255
	d = L.BiasedAttentionDesc()
	for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
		setattr(d, n, p)
	d.B, d.n_head, d.n_kv_head, d.Sq, d.Skv, d.dh, d.dtype = 2, 4, 2, 8, 8, 16, L.BF16
	for n in ("ldq", "ldo", "lddo", "lddq"):
		setattr(d, n, 64)
	for n in ("ldk", "ldv", "lddk", "lddv"):
		setattr(d, n, 32)
	for n in ("batch_q", "batch_o", "batch_do", "batch_dq"):
		setattr(d, n, 512)
	for n in ("batch_k", "batch_v", "batch_dk", "batch_dv"):
		setattr(d, n, 256)
	for n, v in kw.items():
		setattr(d, n, p if v == "p" else v)
	d._keep = buf
	return d


BOTH = [
	(dict(q=None), NULL), (dict(v=None), NULL), (dict(out=None), NULL), (dict(dtype=7), DTYPE), (dict(B=0), SHAPE), (dict(Skv=0), SHAPE), (dict(dh=129), SHAPE), (dict(dh=0), SHAPE),
	(dict(n_kv_head=3), SHAPE), (dict(ldq=63), SHAPE), (dict(ldk=31), SHAPE), (dict(batch_v=-1), SHAPE), (dict(ldv=1 << 40), SHAPE), (dict(Sq=1 << 40), SHAPE), (dict(n_head=1 << 40), SHAPE),
	(dict(softcap=-1.0), SHAPE), (dict(softcap=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE), (dict(q_seg="p"), NULL), (dict(k_pos="p"), NULL), (dict(prefix="p"), UNSUPPORTED),
	(dict(table="p", n_lookup=3, n_bucket=3), NULL), (dict(table="p", lookup="p", n_lookup=0, n_bucket=3), SHAPE), (dict(table="p", lookup="p", n_lookup=3, n_bucket=0), SHAPE),
	(dict(table="p", lookup="p", n_lookup=3, n_bucket=3, lookup_lo=1 << 40), SHAPE), (dict(table="p", lookup="p", n_lookup=3, n_bucket=3), NULL),  # (no prep buffer)
	(dict(table="p", lookup="p", n_lookup=3, n_bucket=3, prep="p", prep_bytes=8), SCRATCH), (dict(q_seg="p", k_seg="p", prep="p", prep_bytes=16), SCRATCH),
]


@pytest.mark.parametrize("kw,code", BOTH)
def test_attention_refuses_at_the_abi(kw, code):
	import vit_amd._lib as L
	lib = L.load()
	d = desc(**kw)
	assert lib.vitk_biased_attention_fwd(d, None) == code
	assert lib.vitk_biased_attention_bwd(d, None) == code


BACKWARD = [(dict(lse=None), NULL), (dict(dk=None), NULL), (dict(dout=None), NULL), (dict(lddq=63), SHAPE), (dict(lddk=31), SHAPE), (dict(batch_dq=0), SHAPE), (dict(batch_dv=31), SHAPE), (dict(dtable="p"), NULL),
	(dict(dtable="p", table="p", lookup="p", n_lookup=3, n_bucket=9000, prep="p", prep_bytes=1 << 20), UNSUPPORTED), (dict(), NULL), (dict(workspace="p", workspace_bytes=16), SCRATCH)]


@pytest.mark.parametrize("kw,code", BACKWARD)
def test_attention_backward_refuses_at_the_abi(kw, code):
	import vit_amd._lib as L
	assert L.load().vitk_biased_attention_bwd(desc(**kw), None) == code


def test_attention_sizes():
	import vit_amd._lib as L
	lib = L.load()
	assert lib.vitk_biased_attention_fwd(None, None) == NULL and lib.vitk_biased_attention_bwd(None, None) == NULL
	assert lib.vitk_biased_attention_prep_bytes(None) == NULL and lib.vitk_biased_attention_workspace_bytes(None, 1) == NULL
	assert lib.vitk_biased_attention_prep_bytes(desc()) == 0 and lib.vitk_biased_attention_workspace_bytes(desc(), 0) == 0
	assert lib.vitk_biased_attention_prep_bytes(desc(dh=200)) == SHAPE and lib.vitk_biased_attention_workspace_bytes(desc(B=-1), 1) == SHAPE
	assert lib.vitk_biased_attention_prep_bytes(desc(table="p", lookup="p", n_lookup=100, n_bucket=3)) >= 4 * 4 * 100
	long = desc(Sq=1, Skv=100000)  # the keys are divided: (max, sum, out) of every part
	assert lib.vitk_biased_attention_workspace_bytes(long, 0) >= 2 * 2 * 4 * 18 * 4
	assert lib.vitk_biased_attention_fwd(long, None) == NULL  # and that needs a workspace


GN = dict(x="p", gamma="p", beta="p", y="p", mean="p", rstd="p", B=2, S=4, C=16, G=4, eps=1e-5, act=2, dtype=1)
GN_BAD = [(dict(x=None), NULL), (dict(y=None), NULL), (dict(mean=None), NULL), (dict(B=0), SHAPE), (dict(S=0), SHAPE), (dict(C=18), SHAPE), (dict(G=0), SHAPE), (dict(B=70000), SHAPE), (dict(C=8192), SHAPE),
	(dict(act=9), UNSUPPORTED), (dict(act=-1), UNSUPPORTED), (dict(dtype=3), DTYPE), (dict(x="odd"), ALIGN), (dict(S=100000, C=256), SCRATCH)]


@pytest.mark.parametrize("kw,code", GN_BAD)
def test_group_norm_refuses_at_the_abi(kw, code):
	import vit_amd._lib as L
	lib = L.load()
	buf = ctypes.create_string_buffer(4096)
	p = (ctypes.addressof(buf) + 255) & ~255
	a = {n: p if v == "p" else p + 1 if v == "odd" else v for n, v in dict(GN, **kw).items()}
	assert lib.vitk_group_norm_fwd(a["x"], a["gamma"], a["beta"], a["y"], a["mean"], a["rstd"], a["B"], a["S"], a["C"], a["G"], a["eps"], a["act"], a["dtype"], None, 0, None) == code
	rc = lib.vitk_group_norm_bwd(a["x"], a["x"], a["gamma"], a["beta"], a["mean"], a["rstd"], a["y"], p, p, 0, a["B"], a["S"], a["C"], a["G"], a["act"], a["dtype"], None, 0, None)
	assert rc == code
	if code == SHAPE:
		assert lib.vitk_group_norm_workspace_bytes(a["B"], a["S"], a["C"], a["G"], a["dtype"]) == SHAPE


def test_group_norm_workspace_is_enough_for_either_direction():
	import vit_amd._lib as L
	lib = L.load()
	for B, S, C, G in ((1, 1, 1, 1), (2, 49, 384, 32), (64, 12544, 256, 32), (300, 7, 16, 2), (1, 1 << 22, 8, 1), (65535, 3, 8, 8)):
		for dt in (0, 1):
			assert lib.vitk_group_norm_workspace_bytes(B, S, C, G, dt) >= 8 * B * C


def test_python_refuses_cpu_tensors_and_bad_arguments():
	from vit_amd import ops
	x = torch.randn(2, 8, 32)
	with pytest.raises(RuntimeError, match="no CPU fallback"):
		ops.biased_attention(x, x, x, 2)
	with pytest.raises(RuntimeError, match="no CPU fallback"):
		ops.group_norm_act(x, None, None, 4)
	with pytest.raises(ValueError, match="activation"):
		ops.group_norm_act(x, None, None, 4, act="tanh")
	i32 = torch.arange(5, dtype=torch.int32)
	with pytest.raises(ValueError, match="together"):
		ops.RelativeBuckets(i32, 0, q_pos=i32)
	with pytest.raises(TypeError, match="int32"):
		ops.RelativeBuckets(i32.long(), 0)
	with pytest.raises(ValueError):
		ops.RelativeBuckets(i32[:0], 0)
	for n, far in ((2, 10), (7, 100), (32, 8)):
		with pytest.raises(ValueError, match="log_distance"):
			ops.RelativeBuckets.log_distance(n, far, "cpu")


def test_module_configurations():
	from vit_amd.layers import RelativeMHA
	from vit_amd.layers.conv import MBConv

	class Cfg:
		d_model, n_head, dropout = 64, 4, 0.0
	m = RelativeMHA(Cfg())
	assert m.rel_bias is None and sorted(m.state_dict()) == ["out_proj.bias", "out_proj.weight", "qkv_proj.weight"]

	class Grid(Cfg):
		attn_grid, n_kv_head = (3, 5), 2
	m = RelativeMHA(Grid())
	assert m.rel_bias.shape == (45, 4) and m.qkv_proj.weight.shape == (64 + 2 * 2 * 16, 64)

	class Both(Grid):
		attn_buckets = (32, 128)
	with pytest.raises(ValueError):
		RelativeMHA(Both())

	class Odd(Cfg):
		n_kv_head = 3
	with pytest.raises(ValueError):
		RelativeMHA(Odd())
	b = MBConv(8, 8, norm_groups=4)
	assert not any("running" in k for k in b.state_dict()) and b.state_dict()["conv.1.weight"].shape == (32,)
	assert any("running_mean" in k for k in MBConv(8, 8).state_dict())


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(gpu):
	from vit_amd import ops
	x = torch.randn(2, 8, 32, device=gpu)
	f = lambda *a, **k: ops.biased_attention(*a, **k)
	i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)
	pl = ops.RelativeBuckets(i32(5), 0)
	for bad, exc in (
		(lambda: f(x, x, x, 5), ValueError), (lambda: f(x, x, x, 4, n_kv_head=3), ValueError), (lambda: f(x, x[:1], x, 4), ValueError), (lambda: f(x[0], x, x, 4), ValueError),
		(lambda: f(torch.randn(1, 4, 260, device=gpu), *[torch.randn(1, 4, 260, device=gpu)] * 2, 2), ValueError), (lambda: f(x, x, x, 4, softcap=-1.0), ValueError),
		(lambda: f(x, x, x, 4, table=torch.randn(5, 4, device=gpu)), ValueError), (lambda: f(x, x, x, 4, table=torch.randn(5, 3, device=gpu), buckets=pl), ValueError),
		(lambda: f(x, x, x, 4, slopes=torch.randn(3, device=gpu)), ValueError), (lambda: f(x, x, x, 4, slopes=torch.randn(4, device=gpu, requires_grad=True)), NotImplementedError),
		(lambda: f(x, x, x, 4, prefix=i32(2)), ValueError), (lambda: f(x, x, x, 4, causal=True, prefix=i32(3)), ValueError), (lambda: f(x, x, x, 4, segments=i32(2, 7)), ValueError),
		(lambda: f(x, x, x, 4, segments=i32(2, 8).long()), TypeError), (lambda: f(x.half(), x.half(), x.half(), 4), TypeError),
		(lambda: f(x, x, x, 4, table=torch.randn(5, 4, device=gpu), buckets=ops.RelativeBuckets(i32(5), 0, i32(7), i32(8))), ValueError),
		(lambda: f(x, x, x, 4, segments=(i32(2, 8), i32(2, 8).cpu())), RuntimeError),
		(lambda: ops.group_norm_act(x, None, None, 5), ValueError), (lambda: ops.group_norm_act(x, torch.ones(31, device=gpu), None, 4), ValueError), (lambda: ops.group_norm_act(x[0], None, None, 4), ValueError),
	):
		with pytest.raises(exc):
			bad()
	t = torch.randn(9000, 4, device=gpu, requires_grad=True)  # more buckets than the gradient's sums hold; without a gradient it is fine
	with pytest.raises(ValueError, match="8192"):
		f(x, x, x, 4, table=t, buckets=pl)
	assert f(x, x, x, 4, table=t.detach(), buckets=pl).shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-1.0, 0.0, float("nan"), float("inf")])
def test_a_scale_that_is_not_positive_is_refused(gpu, scale):
	from vit_amd import ops
	x = torch.zeros(1, 4, 16, device=gpu)
	with pytest.raises(ValueError, match="scale"):
		ops.biased_attention(x, x, x, 1, scale=scale)


def test_divided_keys_with_an_odd_head_size():
	"""One query of one head of 7 columns, 11 tiles of keys in 3 parts: 21 sums, and the three pairs behind them begin at the next even float."""
	import vit_amd._lib as L
	lib = L.load()
	d = desc(B=1, n_head=1, n_kv_head=1, Sq=1, Skv=11 * 64, dh=7, workspace="p", workspace_bytes=(21 + 6) * 4)
	assert lib.vitk_biased_attention_workspace_bytes(d, 0) >= (22 + 6) * 4
	assert lib.vitk_biased_attention_fwd(d, None) == SCRATCH


@pytest.mark.parametrize("kind", [dict(attn_grid=(3, 5)), dict(attn_buckets=(8, 20))])
def test_buckets_made_in_inference_mode_serve_training(kind):
	"""RelativeMHA keeps its buckets from the first forward on: tensors made in inference mode cannot be saved for a backward."""
	from vit_amd.layers import RelativeMHA
	m = RelativeMHA(type("Cfg", (), dict(d_model=64, n_head=4, dropout=0.0, **kind))())
	with torch.inference_mode():
		b = m.buckets(torch.device("cpu"))
	assert b is m.buckets(torch.device("cpu"))
	assert not any(t.is_inference() for t in (b.lookup, b.q_pos, b.k_pos) if t is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(gpu, grad):
	"""Neither operator has them: a dual tensor among the operands is an error, not a result without its tangent."""
	import torch.autograd.forward_ad as ad
	from vit_amd import ops
	x, t, s = torch.randn(1, 4, 16, device=gpu), torch.randn(5, 2, device=gpu), torch.randn(2, device=gpu)
	pl = ops.RelativeBuckets(torch.zeros(5, dtype=torch.int32, device=gpu), 0)
	w = torch.ones(16, device=gpu)
	with ad.dual_level(), torch.set_grad_enabled(grad):
		dual = lambda a: ad.make_dual(a, torch.ones_like(a))
		for call in (lambda: ops.biased_attention(dual(x), x, x, 2), lambda: ops.biased_attention(x, x, dual(x), 2), lambda: ops.biased_attention(x, x, x, 2, table=dual(t), buckets=pl),
			lambda: ops.biased_attention(x, x, x, 2, slopes=dual(s)), lambda: ops.group_norm_act(dual(x), w, w, 4), lambda: ops.group_norm_act(x, w, dual(w), 4)):
			with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
				call()
		assert ops.biased_attention(x, x, x, 2, slopes=s).shape == ops.group_norm_act(x, w, w, 4).shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("rows", [0, 4])
def test_group_norm_refuses_other_types(gpu, dtype, rows):
	"""Of float16 and float64 an empty batch came back as float32 (any other was refused)."""
	from vit_amd import ops
	with pytest.raises(TypeError, match="float32 and bfloat16"):
		ops.group_norm_act(torch.zeros(rows, 3, 8, dtype=dtype, device=gpu), None, None, 2)


def test_rows_far_apart_are_copied():
	"""The kernels reach rows that lie up to 2^21 elements apart."""
	from vit_amd import ops
	far = torch.empty_strided((1, 2, 8), (8, (1 << 21) + 8, 1), device="meta")
	assert ops._rows_of(far, 8).stride() == (16, 8, 1)
	near = torch.empty_strided((1, 2, 8), (8, 1 << 21, 1), device="meta")
	assert ops._rows_of(near, 8) is near
	one = torch.empty_strided((3, 1, 8), (8, 1 << 40, 1), device="meta")
	assert ops._rows_of(one, 8) is one


@pytest.mark.gpu
def test_slopes_that_could_take_a_gradient_serve_evaluation(gpu):
	from vit_amd import ops
	x, s = torch.randn(1, 6, 16, device=gpu), torch.nn.Parameter(torch.tensor([0.5, 0.25], device=gpu))
	with pytest.raises(NotImplementedError, match="slopes"):
		ops.biased_attention(x, x, x, 2, slopes=s)
	with torch.no_grad():
		y = ops.biased_attention(x, x, x, 2, slopes=s)
	assert torch.equal(y, ops.biased_attention(x, x, x, 2, slopes=s.detach()))


@pytest.mark.parametrize("kw", [dict(batch_qpos=-1), dict(batch_kpos=-8)])
def test_negative_strides_of_positions_are_refused(kw):
	import vit_amd._lib as L
	lib = L.load()
	d = desc(q_pos="p", k_pos="p", slopes="p", prep="p", prep_bytes=0, **kw)
	assert lib.vitk_biased_attention_prep_bytes(d) == SHAPE and lib.vitk_biased_attention_workspace_bytes(d, 1) == SHAPE
	assert lib.vitk_biased_attention_fwd(d, None) == SHAPE and lib.vitk_biased_attention_bwd(d, None) == SHAPE


def test_mbconv_asks_for_like_group_norms():
	"""Its three norms run with one eps and one number of groups: others set on a module are an error, as with BatchNorm."""
	from vit_amd.layers.conv import MBConv
	for name, value in (("eps", 1e-3), ("num_groups", 2)):
		m = MBConv(8, 8, norm_groups=4)
		setattr(m.conv[4], name, value)
		with pytest.raises(AssertionError):
			m(torch.zeros(1, 8, 4, 4))


def test_prep_holds_the_rest_of_out():
	import vit_amd._lib as L
	lib = L.load()
	assert L.BiasedAttentionDesc.keep_rest.offset == ctypes.sizeof(L.BiasedAttentionDesc) - 4
	assert lib.vitk_biased_attention_prep_bytes(desc(keep_rest=1)) >= 2 * 2 * 8 * 64 and lib.vitk_biased_attention_prep_bytes(desc(keep_rest=1, dtype=L.F32)) == 0
	assert lib.vitk_biased_attention_fwd(desc(keep_rest=1), None) == NULL and lib.vitk_biased_attention_bwd(desc(keep_rest=1), None) == NULL
	assert lib.vitk_biased_attention_fwd(desc(keep_rest=1, prep="p", prep_bytes=2047), None) == SCRATCH
