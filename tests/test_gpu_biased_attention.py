"""GPU: attention with bucket bias, distance slopes, tanh cap, segments and causal prefix masks (ops.biased_attention) against a plain
float64 evaluation of its definition on the same inputs, element by element.

Tolerances, from the arithmetic (u = half a step of the storage type, 2^-8 for bfloat16 and 2^-24 for float32; f = 2e-5):
  * every float32 quantity carries a relative error below f: scores are at most about 64 in units of log2 here, a step of which is 4e-6,
    and p = 2^(z - m) turns that into as much relative error of p, a few times over; sums add the terms' errors, so f multiplies the sum of
    the terms' absolute values;
  * bfloat16: each product's weights (p, dz) are rounded once, at most u of each term, and the result once, u of itself; delta = rowsum(dout o out)
    comes from a rounded out that itself carries u (|out| + p |v|), so each dz also carries p u sum_d |dout| (2 |out| + p |v|).
The table gradient has float32 arithmetic throughout, with either operand type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F = 2e-5
U = {torch.bfloat16: 2.0 ** -8, torch.float32: F}


def make(B, H, Hkv, Sq, Skv, dh, dtype, seed=0, gain=1.0, requires=True):
	g = torch.Generator().manual_seed(seed)
	mk = lambda S, h, k=1.0: (k * torch.randn(B, S, h * dh, generator=g)).to(dtype)
	return mk(Sq, H, gain), mk(Skv, Hkv), mk(Skv, Hkv), mk(Sq, H)


def visible(B, Sq, Skv, segments=None, causal=False, prefix=None):
	vis = torch.ones(B, Sq, Skv, dtype=torch.bool)
	if segments is not None:
		qs, ks = segments
		vis &= (qs[:, :, None] == ks[:, None, :]) & (ks[:, None, :] >= 0)
	if causal:
		i, j = torch.arange(Sq)[:, None] + Skv - Sq, torch.arange(Skv)[None]
		seen = (j <= i)[None]
		if prefix is not None:
			seen = seen | (j[None] < prefix[:, None, None])
		vis &= seen
	return vis


def reference(q, k, v, dout, H, Hkv, scale=None, softcap=0.0, table=None, lookup=None, lo=0, q_pos=None, k_pos=None, slopes=None, **mask):
	"""(values, bounds) of out, dq, dk, dv and dtable in float64; hidden pairs contribute nothing whatever they hold."""
	B, Sq, _ = q.shape
	Skv, dh = k.shape[1], q.shape[2] // H
	scale = scale or dh ** -0.5
	heads = lambda t, n: t.double().view(B, -1, n, dh).transpose(1, 2)
	Q, K, V, G = heads(q, H), heads(k, Hkv).repeat_interleave(H // Hkv, 1), heads(v, Hkv).repeat_interleave(H // Hkv, 1), heads(dout, H)
	vis = visible(B, Sq, Skv, **mask)[:, None]
	# rows and keys of no visible pair are taken as zero: they may hold anything
	rows, keys = vis.any(3), vis.any(2)
	Q, G = (torch.where(rows[..., None], t, 0.0) for t in (Q, G))
	K, V = (torch.where(keys[..., None], t, 0.0) for t in (K, V))
	s = Q @ K.transpose(2, 3) * scale
	t = torch.tanh(s / softcap) if softcap else None
	z = softcap * t if softcap else s
	qp = (q_pos if q_pos is not None else torch.arange(Sq) + Skv - Sq).long()
	kp = (k_pos if k_pos is not None else torch.arange(Skv)).long()
	qp, kp = (p if p.dim() == 2 else p[None] for p in (qp, kp))
	d = kp[:, None, :] - qp[:, :, None]
	if table is not None:
		idx = (d - lo).clamp(0, lookup.numel() - 1)
		bucket = lookup.long()[idx]
		ok = (bucket >= 0) & (bucket < table.shape[0])
		z = z + torch.where(ok[..., None], table.double()[bucket.clamp(0, table.shape[0] - 1)], 0.0).permute(0, 3, 1, 2)
	if slopes is not None:
		z = z - slopes.double()[None, :, None, None] * d.abs()[:, None].double()
	z = z.masked_fill(~vis, -math.inf)
	m = z.amax(-1, keepdim=True)
	e = torch.exp(z - torch.where(m.isinf(), 0.0, m))
	l = e.sum(-1, keepdim=True)
	p = e / torch.where(l == 0, 1.0, l)
	u = U[q.dtype]
	merge = lambda x, n: x.transpose(1, 2).reshape(B, -1, n * dh)
	share = lambda x: x.view(B, Hkv, H // Hkv, Skv, dh).sum(2)
	val, tol = {}, {}
	out, pv = p @ V, p @ V.abs()
	val["out"], tol["out"] = merge(out, H), merge(u * (out.abs() + pv) + F * pv, H)
	dv, dva = p.transpose(2, 3) @ G, p.transpose(2, 3) @ G.abs()
	val["dv"], tol["dv"] = merge(share(dv), Hkv), merge((u + F) * share(dva) + u * share(dv).abs(), Hkv)
	dp, dpa = G @ V.transpose(2, 3), G.abs() @ V.abs().transpose(2, 3)
	delta = (p * dp).sum(-1, keepdim=True)
	dz = p * (dp - delta)
	de = (G.abs() * (u * (2 * out.abs() + pv) + F * pv)).sum(-1, keepdim=True)  # error of delta
	fine = F * p * (dpa + (p * dpa).sum(-1, keepdim=True))
	if table is not None:
		w = torch.zeros(table.shape[0], H, dtype=torch.float64)
		wt = torch.zeros_like(w)
		for b in range(B):
			bb = bucket[b if bucket.shape[0] > 1 else 0]
			good = ok[b if ok.shape[0] > 1 else 0]
			for h in range(H):
				w[:, h].index_add_(0, bb[good], dz[b, h][good])
				wt[:, h].index_add_(0, bb[good], fine[b, h][good])
		val["dtable"], tol["dtable"] = w, wt + 1e-30
	edz = u * dz.abs() + p * de + fine
	if softcap:
		dz, edz = dz * (1 - t * t), edz * (1 - t * t) + F * dz.abs()
	val["dq"], tol["dq"] = merge(dz @ K * scale, H), merge(edz @ K.abs() * scale, H)
	dk = share(dz.transpose(2, 3) @ Q * scale)
	val["dk"], tol["dk"] = merge(dk, Hkv), merge(share(edz.transpose(2, 3) @ Q.abs() * scale), Hkv)
	for n in ("dq", "dk"):
		tol[n] = tol[n] + u * val[n].abs()
	return val, tol


def run(gpu, q, k, v, dout, H, Hkv, table=None, lookup=None, lo=0, q_pos=None, k_pos=None, slopes=None, segments=None, prefix=None, **kw):
	from vit_amd import ops
	dev = lambda t: t.to(gpu) if t is not None else None
	leaves = [dev(t).requires_grad_() for t in (q, k, v)]
	tb = dev(table).requires_grad_() if table is not None else None
	buckets = ops.RelativeBuckets(dev(lookup), lo, dev(q_pos), dev(k_pos)) if table is not None else None
	out = ops.biased_attention(*leaves, H, n_kv_head=Hkv, table=tb, buckets=buckets, slopes=dev(slopes), segments=tuple(dev(t) for t in segments) if segments is not None else None,
		prefix=dev(prefix), **kw)
	grads = torch.autograd.grad(out, leaves + ([tb] if tb is not None else []), dev(dout))
	return dict(zip(["out", "dq", "dk", "dv", "dtable"], [out.detach(), *grads]))


def check(got, val, tol):
	for n, x in got.items():
		a, b, t = x.double().cpu(), val[n], tol[n]
		assert a.shape == b.shape and torch.isfinite(a).all(), n
		worst = ((a - b).abs() / (t + 1e-12)).max().item()
		assert worst <= 1.0, f"{n}: {worst:.2f} times the bound"


def grid_positions(h, w):
	return (torch.arange(h)[:, None] * (2 * w - 1) + torch.arange(w)).reshape(-1).to(torch.int32), torch.arange((2 * h - 1) * (2 * w - 1), dtype=torch.int32), -((h - 1) * (2 * w - 1) + w - 1)


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,dh", [(2, 3, 3, 65, 65, 64), (1, 4, 2, 1, 1, 32), (2, 2, 1, 130, 200, 12), (1, 2, 2, 300, 33, 7), (1, 3, 1, 129, 128, 128), (3, 2, 2, 31, 64, 40), (1, 8, 2, 64, 257, 96), (2, 1, 1, 17, 5, 1), (1, 2, 2, 5, 700, 20)])
def test_plain_softmax_shapes(gpu, dtype, B, H, Hkv, Sq, Skv, dh):
	q, k, v, g = make(B, H, Hkv, Sq, Skv, dh, dtype, seed=Sq + dh)
	check(run(gpu, q, k, v, g, H, Hkv), *reference(q, k, v, g, H, Hkv))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,w,dh,H", [(7, 7, 32, 3), (5, 9, 12, 4), (1, 130, 64, 2), (14, 14, 64, 2), (40, 2, 24, 1), (12, 12, 128, 2)])
def test_grid_bias(gpu, dtype, h, w, dh, H):
	S = h * w
	q, k, v, g = make(3, H, H, S, S, dh, dtype, seed=S)
	pos, lookup, lo = grid_positions(h, w)
	table = torch.randn(lookup.numel(), H, generator=torch.Generator().manual_seed(1))
	kw = dict(table=table, lookup=lookup, lo=lo, q_pos=pos, k_pos=pos)
	check(run(gpu, q, k, v, g, H, H, **kw), *reference(q, k, v, g, H, H, **kw))


def test_grid_helper_is_the_table_layout(gpu):
	"""RelativeBuckets.grid: bucket (dy + h - 1)(2w - 1) + dx + w - 1 of a key dy rows below and dx columns right of the query."""
	from vit_amd import ops
	h, w = 3, 4
	pl = ops.RelativeBuckets.grid(h, w, gpu)
	pos, lookup, lo = pl.k_pos.cpu(), pl.lookup.cpu(), pl.lo
	for i in range(h * w):
		for j in range(h * w):
			dy, dx = j // w - i // w, j % w - i % w
			assert lookup[int(pos[j] - pos[i]) - lo] == (dy + h - 1) * (2 * w - 1) + dx + w - 1
	b = ops.RelativeBuckets.log_distance(32, 128, gpu).lookup.cpu()
	assert b[128] == 0 and b[127] == 1 and b[129] == 17 and b[0] == 15 and b[-1] == 31 and b.max() == 31


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Sq,Skv,dh", [(1, 900, 64), (300, 300, 64), (64, 700, 32), (700, 40, 64), (1, 2500, 128), (16, 1500, 12)])
def test_log_buckets_and_divided_axes(gpu, dtype, Sq, Skv, dh):
	"""Distances far beyond the lookup (one bucket for most of a row, whose gradient nearly cancels), few queries over many keys and many queries
	over few keys (the streamed axis divided among workgroups)."""
	from vit_amd import ops
	H = 2
	q, k, v, g = make(2, H, 1, Sq, Skv, dh, dtype, seed=Skv)
	pl = ops.RelativeBuckets.log_distance(16, 40, "cpu")
	table = torch.randn(16, H, generator=torch.Generator().manual_seed(2))
	kw = dict(table=table, lookup=pl.lookup, lo=pl.lo)
	check(run(gpu, q, k, v, g, H, 1, **kw), *reference(q, k, v, g, H, 1, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["repeated", "wide", "per_image", "no_bucket", "with_slopes"])
def test_positions_of_any_kind(gpu, dtype, kind):
	"""Positions that repeat within a wave (the scatter by distance is not possible), positions whose distances span more than a window, positions of each
	image's own, lookup entries that name no bucket, and a table together with slopes."""
	B, H, S, dh, nb = 2, 2, 140, 32, 37
	g_ = torch.Generator().manual_seed(3)
	q, k, v, g = make(B, H, H, S, S, dh, dtype, seed=4)
	lookup = torch.randint(0, nb, (301,), generator=g_).to(torch.int32)
	lo, slopes = -150, None
	qp = kp = torch.arange(S, dtype=torch.int32)
	if kind == "repeated":
		qp = kp = torch.randint(0, 9, (S,), generator=g_).to(torch.int32)
	elif kind == "wide":
		qp = kp = torch.randint(-100000, 100000, (S,), generator=g_).to(torch.int32)
		lookup, lo = torch.randint(0, nb, (200001,), generator=g_).to(torch.int32), -100000
	elif kind == "per_image":
		qp = torch.stack([torch.randperm(S, generator=g_) for _ in range(B)]).to(torch.int32)
		kp = torch.stack([torch.randperm(S, generator=g_) for _ in range(B)]).to(torch.int32)
	elif kind == "no_bucket":
		lookup = torch.randint(-5, nb + 5, (301,), generator=g_).to(torch.int32)
	else:
		slopes = torch.tensor([0.25, 0.0625])
	table = torch.randn(nb, H, generator=g_)
	kw = dict(table=table, lookup=lookup, lo=lo, q_pos=qp, k_pos=kp, slopes=slopes)
	check(run(gpu, q, k, v, g, H, H, **kw), *reference(q, k, v, g, H, H, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Sq,Skv,prefix", [(65, 65, None), (200, 200, (0, 200)), (130, 300, (7, 150)), (300, 130, (0, 64)), (1, 257, (3, 250)), (5, 3, None)])
@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_causal_prefix_and_cap(gpu, dtype, Sq, Skv, prefix, softcap):
	"""Causal masks aligned at the end (with more queries than keys the first queries see nothing), prefixes of none and all of the keys; a small cap
	puts most scores on the curved part of the tanh."""
	H, dh = 4, 64
	q, k, v, g = make(2, H, 2, Sq, Skv, dh, dtype, seed=5, gain=3.0 if softcap else 1.0)
	mask = dict(causal=True, prefix=torch.tensor(prefix, dtype=torch.int32) if prefix else None)
	check(run(gpu, q, k, v, g, H, 2, softcap=softcap, **mask), *reference(q, k, v, g, H, 2, softcap=softcap, **mask))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["packed", "shuffled", "padding", "none_match"])
@pytest.mark.parametrize("extra", ["", "slopes", "causal"])
def test_segments(gpu, dtype, kind, extra):
	"""Documents behind one another, in no order, with padding of NaN (not read), and queries whose segment no key has."""
	B, H, S, dh = 2, 2, 333, 32
	g_ = torch.Generator().manual_seed(6)
	q, k, v, g = make(B, H, H, S, S, dh, dtype, seed=7)
	seg = (torch.rand(B, S, generator=g_) < 0.02).cumsum(1).to(torch.int32)
	qs, ks = seg, seg
	if kind == "shuffled":
		qs = ks = torch.randint(0, 5, (B, S), generator=g_).to(torch.int32)
	elif kind == "padding":
		qs = ks = torch.where(torch.arange(S) < torch.tensor([[200], [333]]), seg, -7).to(torch.int32)
		for t in (q, k, v, g):
			t[qs < 0] = float("nan")
	elif kind == "none_match":
		ks = seg + 100
	kw = dict(segments=(qs, ks))
	if extra == "slopes":
		kw["slopes"] = torch.tensor([0.5, 0.01])
	if extra == "causal":
		kw["causal"] = True
	got = run(gpu, q, k, v, g, H, H, **kw)
	check(got, *reference(q, k, v, g, H, H, **kw))
	if kind == "none_match":
		assert all(float(x.abs().max()) == 0.0 for x in got.values())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_specials_in_hidden_places(gpu, dtype, value):
	"""A key, value, query or gradient row of one document that holds an infinity or a NaN leaves the other documents alone, within a tile too; keys
	behind every query's causal limit likewise."""
	B, H, S, dh = 1, 2, 150, 64
	q, k, v, g = make(B, H, H, S, S, dh, dtype, seed=8)
	seg = (torch.arange(S) // 50).to(torch.int32)[None]
	kw = dict(segments=(seg, seg))
	val, tol = reference(q, k, v, g, H, H, **kw)
	for t in (q, k, v, g):
		t[0, 70] = value  # document 1
	got = run(gpu, q, k, v, g, H, H, **kw)
	other = (seg[0] != 1).nonzero()[:, 0]
	for n, x in got.items():
		a = x.double().cpu()[:, other]
		assert torch.isfinite(a).all(), n
		assert ((a - val[n][:, other]).abs() <= tol[n][:, other] + 1e-12).all(), n
	# queries 0 .. 69 see keys 0 .. 69 at most: 100 keys hold `value` behind them
	q, k, v, g = make(B, H, H, S, S, dh, dtype, seed=9)
	k[0, 120:], v[0, 120:] = value, value
	out = run(gpu, q, k, v, g, H, H, causal=True)["out"].cpu()
	assert torch.isfinite(out[0, :120].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_class_rows(gpu, dtype):
	"""q, k, v as column slices of one joint buffer, the class-token row alone as query (a batch stride that is not rows * row stride), keys broadcast over
	the batch, and a transposed buffer whose rows are not contiguous."""
	from vit_amd import ops
	B, S, H, dh = 3, 77, 2, 24
	d = H * dh
	g_ = torch.Generator().manual_seed(10)
	qkv = torch.randn(B, S, 3 * d, generator=g_).to(dtype)
	g = torch.randn(B, S, d, generator=g_).to(dtype)
	joint = qkv.to(gpu).requires_grad_()
	out = ops.biased_attention(joint[..., :d], joint[..., d:2 * d], joint[..., 2 * d:], H, causal=True)
	(dj,) = torch.autograd.grad(out, joint, g.to(gpu))
	val, tol = reference(*qkv.split(d, 2), g, H, H, causal=True)
	check({"out": out.detach(), "dq": dj[..., :d], "dk": dj[..., d:2 * d], "dv": dj[..., 2 * d:]}, val, tol)
	with torch.no_grad():
		dev = qkv.to(gpu)
		one = ops.biased_attention(dev[:, :1, :d], dev[..., d:2 * d], dev[..., 2 * d:], H)
		val, tol = reference(qkv[:, :1, :d], qkv[..., d:2 * d], qkv[..., 2 * d:], g[:, :1], H, H)
		check({"out": one}, val, tol)
		wide = ops.biased_attention(dev[..., :d], dev[:1, :, d:2 * d].expand(B, S, d), dev[:1, :, 2 * d:].expand(B, S, d), H)
		val, tol = reference(qkv[..., :d], qkv[:1, :, d:2 * d].expand(B, S, d), qkv[:1, :, 2 * d:].expand(B, S, d), g, H, H)
		check({"out": wide}, val, tol)
		flip = dev[..., :d].transpose(1, 2).contiguous().transpose(1, 2)
		val, tol = reference(qkv[..., :d], qkv[..., d:2 * d], qkv[..., 2 * d:], g, H, H)
		check({"out": ops.biased_attention(flip, dev[..., d:2 * d], dev[..., 2 * d:], H)}, val, tol)
		odd = torch.empty(B * S * d + 1, dtype=dtype, device=gpu)[1:].view(B, S, d)  # not 16-byte aligned
		odd.copy_(dev[..., :d])
		check({"out": ops.biased_attention(odd, dev[..., d:2 * d], dev[..., 2 * d:], H)}, val, tol)


def test_gradients_against_differences(gpu):
	"""Central differences of <out, dout> in float32 along random directions: with steps h = 2^-6 the curvature term is O(h^2) of a smooth function of unit
	size (2.5e-4 times a third derivative of a few units) and the rounding term 2^-24 * |<out, dout>| / h, about 4e-5 * |..|: 1 % covers both."""
	from vit_amd import ops
	B, H, S, dh = 2, 2, 40, 16
	g_ = torch.Generator().manual_seed(11)
	q, k, v, g = (t.to(gpu) for t in make(B, H, H, S, S, dh, torch.float32, seed=12))
	pl = ops.RelativeBuckets.grid(5, 8, gpu)
	table = (0.5 * torch.randn(pl.lookup.numel(), H, generator=g_)).to(gpu)
	seg = (torch.arange(S, device=gpu) // 25).to(torch.int32).expand(B, S).contiguous()
	f = lambda q, k, v, t: ops.biased_attention(q, k, v, H, table=t, buckets=pl, softcap=2.0, segments=seg)
	xs = [t.clone().requires_grad_() for t in (q, k, v, table)]
	grads = torch.autograd.grad(f(*xs), xs, g)
	for n in range(4):
		e = torch.randn(xs[n].shape, generator=g_).to(gpu)
		h = 2.0 ** -6
		with torch.no_grad():
			at = lambda s: (f(*[x + s * h * e if i == n else x for i, x in enumerate(xs)]).double() * g.double()).sum()
			num = float((at(1) - at(-1)) / (2 * h))
		ana = float((grads[n].double() * e.double()).sum())
		assert abs(num - ana) < 1e-2 * max(abs(num), float(grads[n].double().norm())), (n, num, ana)


def test_same_bits_every_time_and_on_another_stream(gpu):
	q, k, v, g = make(4, 4, 2, 196, 196, 64, torch.bfloat16, seed=13)
	pos, lookup, lo = grid_positions(14, 14)
	kw = dict(table=torch.randn(lookup.numel(), 4, generator=torch.Generator().manual_seed(1)), lookup=lookup, lo=lo, q_pos=pos, k_pos=pos)
	first = run(gpu, q, k, v, g, 4, 2, **kw)
	s = torch.cuda.Stream()
	for i in range(3):
		with torch.cuda.stream(s if i == 1 else torch.cuda.current_stream()):
			again = run(gpu, q, k, v, g, 4, 2, **kw)
		torch.cuda.synchronize()
		for n in first:
			assert torch.equal(first[n], again[n]), n


def test_captured_step_replays(gpu):
	"""Forward and backward in a HIP graph, replayed with new inputs between eager calls and synchronisations: every replay equals the eager result."""
	from vit_amd import ops
	B, S, H, dh = 2, 130, 2, 64
	pl = ops.RelativeBuckets.log_distance(16, 40, gpu)
	sets = [[t.to(gpu) for t in make(B, H, H, S, S, dh, torch.bfloat16, seed=20 + i)] for i in range(3)]
	seg = (torch.arange(S, device=gpu) // 50).to(torch.int32).expand(B, S).contiguous()
	table0 = torch.randn(16, H, device=gpu)

	def step(q, k, v, g, t):
		out = ops.biased_attention(q, k, v, H, table=t, buckets=pl, segments=seg, softcap=10.0)
		return [out.detach(), *torch.autograd.grad(out, (q, k, v, t), g)]

	eager = [step(*(t.clone().requires_grad_() for t in s[:3]), s[3], table0.clone().requires_grad_()) for s in sets]
	static = [t.clone().requires_grad_() for t in sets[0][:3]] + [sets[0][3].clone(), table0.clone().requires_grad_()]
	side = torch.cuda.Stream()
	side.wait_stream(torch.cuda.current_stream())
	with torch.cuda.stream(side):
		for _ in range(2):
			step(*static)
	torch.cuda.current_stream().wait_stream(side)
	torch.cuda.synchronize()
	graph = torch.cuda.CUDAGraph()
	with torch.cuda.graph(graph):
		res = step(*static)
	for i in (0, 1, 2, 1):
		with torch.no_grad():
			for dst, src in zip(static[:4], sets[i]):
				dst.copy_(src)
		graph.replay()
		torch.cuda.synchronize()
		for a, b in zip(res, eager[i]):
			assert torch.equal(a, b), i
		torch.randn(1000, device=gpu).sum().item()


@pytest.mark.parametrize("B,Sq,Skv", [(0, 4, 4), (2, 0, 4), (2, 3, 0)])
def test_nothing_to_attend(gpu, B, Sq, Skv):
	from vit_amd import ops
	q, k, v = (torch.randn(B, S, 32, device=gpu).requires_grad_() for S in (Sq, Skv, Skv))
	out = ops.biased_attention(q, k, v, 2)
	assert out.shape == q.shape and float(out.detach().abs().sum()) == 0.0
	for t in torch.autograd.grad(out.sum(), (q, k, v)):
		assert float(t.abs().sum()) == 0.0


def test_long_cache_offsets(gpu):
	"""Rows whose byte offsets pass 2^31: one query over a cache of 2.2 GB, whose last rows alone are visible."""
	from vit_amd import ops
	S, H, dh = 1_200_000, 7, 128
	k = torch.zeros(1, S, H * dh, dtype=torch.bfloat16, device=gpu)
	v = torch.zeros_like(k)
	q = torch.randn(1, 1, H * dh, device=gpu).bfloat16()
	tail = torch.randn(1, 5, H * dh, device=gpu).bfloat16()
	k[:, -5:], v[:, -5:] = tail, tail.flip(1)
	seg = torch.full((1, S), -1, dtype=torch.int32, device=gpu)
	seg[:, -5:] = 0
	with torch.no_grad():
		out = ops.biased_attention(q, k, v, H, segments=(torch.zeros(1, 1, dtype=torch.int32, device=gpu), seg))
		want = ops.biased_attention(q, tail, tail.flip(1), H)
	val, tol = reference(q.cpu(), tail.cpu(), tail.flip(1).cpu(), q.cpu(), H, H)
	check({"out": out}, val, tol)
	check({"out": want}, val, tol)


def test_mixed_types_and_autocast(gpu):
	"""Under bf16 autocast float32 operands are computed in bfloat16 and their gradients come back in float32."""
	from vit_amd import ops
	q, k, v, g = (t.to(gpu) for t in make(2, 2, 2, 50, 50, 32, torch.float32, seed=14))
	leaves = [t.requires_grad_() for t in (q, k, v)]
	with torch.autocast("cuda", dtype=torch.bfloat16):
		out = ops.biased_attention(*leaves, 2)
	assert out.dtype == torch.bfloat16
	grads = torch.autograd.grad(out, leaves, g.bfloat16())
	assert all(t.dtype == torch.float32 for t in grads)
	val, tol = reference(*(t.detach().bfloat16().cpu() for t in (q, k, v, g)), 2, 2)
	check(dict(zip(("out", "dq", "dk", "dv"), [out.detach(), *grads])), val, tol)


def test_gradient_sink_of_the_table(gpu):
	"""A table with a registered gradient sink: its gradient is added there, and autograd gets none."""
	from vit_amd import ops
	q, k, v, g = (t.to(gpu) for t in make(2, 2, 2, 49, 49, 32, torch.bfloat16, seed=15))
	pl = ops.RelativeBuckets.grid(7, 7, gpu)
	table = torch.nn.Parameter(torch.randn(169, 2, device=gpu))
	f = lambda: ops.biased_attention(q.requires_grad_(), k, v, 2, table=table, buckets=pl)
	(want,) = torch.autograd.grad(f(), table, g)
	buf = torch.ones_like(table)
	ops.register_grad_sink(table, buf)
	try:
		f().backward(g)
	finally:
		ops.unregister_grad_sink(table)
	assert table.grad is None and torch.equal(buf, want + 1.0)


def test_masks_changed_before_the_backward_are_noticed(gpu):
	"""The forward leaves ranges of the segments and positions for the backward: changing those in place in between is an error, not a wrong gradient."""
	from vit_amd import ops
	q, k, v, g = (t.to(gpu) for t in make(1, 2, 2, 64, 64, 32, torch.bfloat16, seed=16))
	seg = torch.zeros(1, 64, dtype=torch.int32, device=gpu)
	out = ops.biased_attention(q.requires_grad_(), k, v, 2, segments=seg)
	seg[:, 32:] = 1
	with pytest.raises(RuntimeError, match="modified by an inplace operation"):
		out.backward(g)


@pytest.mark.parametrize("kind", ["bf16", "strided"])
def test_table_of_another_type_is_read_at_each_replay(gpu, kind):
	"""A table that the kernels cannot read as it is gets copied at every call, inside a captured one too."""
	from vit_amd import ops
	q, k, v, _ = (t.to(gpu) for t in make(1, 2, 2, 49, 49, 32, torch.bfloat16, seed=17))
	pl = ops.RelativeBuckets.grid(7, 7, gpu)
	table = torch.randn(169, 2, device=gpu).bfloat16() if kind == "bf16" else torch.randn(169, 4, device=gpu)[:, ::2]
	f = lambda: ops.biased_attention(q, k, v, 2, table=table, buckets=pl)
	f()
	side = torch.cuda.Stream()
	side.wait_stream(torch.cuda.current_stream())
	with torch.cuda.stream(side):
		f()
	torch.cuda.current_stream().wait_stream(side)
	graph = torch.cuda.CUDAGraph()
	with torch.cuda.graph(graph):
		out = f()
	for i in range(3):
		table.copy_(torch.randn(169, 2, device=gpu))
		graph.replay()
		torch.cuda.synchronize()
		assert torch.equal(out, f()), i


def test_without_gradient_the_bits_are_the_same(gpu):
	from vit_amd import ops
	q, k, v, _ = (t.to(gpu) for t in make(2, 2, 2, 70, 90, 40, torch.bfloat16, seed=18))
	want = ops.biased_attention(q.requires_grad_(), k, v, 2, causal=True)
	assert want.requires_grad
	with torch.no_grad():
		out = ops.biased_attention(q, k, v, 2, causal=True)
	assert not out.requires_grad and torch.equal(out, want)


@pytest.mark.parametrize("dh", [12, 64, 80, 128])
@pytest.mark.parametrize("kind", ["one token", "one token sloped", "one token capped", "documents of one token", "prefix"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_that_sees_one_key_has_no_score_gradient(gpu, dtype, kind, dh):
	"""A softmax over one key is 1 whatever the score: out is the value, dq and dk are exactly 0, dv is the gradient."""
	from vit_amd import ops
	S = 1 if kind.startswith("one") else 70
	q, k, v, g = (t.to(gpu) for t in make(3, 2, 2, S, S, dh, dtype, seed=19))
	kw = dict(softcap=30.0) if kind != "one token" else {}
	if kind == "one token sloped":
		kw = dict(slopes=torch.ones(2, device=gpu))
	if kind.startswith("documents"):
		kw["segments"] = torch.arange(S, dtype=torch.int32, device=gpu).expand(3, S)
	if kind == "prefix":  # a causal mask's first row: the rows behind it get no gradient here
		kw.update(causal=True)
		g[:, 1:] = 0
	leaves = [t.requires_grad_() for t in (q, k, v)]
	out = ops.biased_attention(*leaves, 2, **kw)
	dq, dk, dv = torch.autograd.grad(out, leaves, g)
	n = S if kind != "prefix" else 1
	assert torch.equal(out[:, :n], v[:, :n])
	# (the weight 2^(s - lse) takes s from the product and lse from the forward, which rounded s * scale: for |s| < 64 an error below 64 * 2^-24)
	assert float((dv - g).abs().max()) <= 2.0 ** -18 * float(g.abs().max())
	assert float(dq.abs().max()) == 0.0 and float(dk.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Sq,Skv,dh", [(1, 1, 1, 700, 7), (1, 3, 5, 1500, 1), (3, 1, 1, 900, 33)])
def test_divided_keys_with_an_odd_head_size(gpu, dtype, B, H, Sq, Skv, dh):
	"""An odd number of rows, parts and columns: what the parts leave is not a whole number of pairs."""
	q, k, v, g = make(B, H, H, Sq, Skv, dh, dtype, seed=Skv)
	check(run(gpu, q, k, v, g, H, H), *reference(q, k, v, g, H, H))


def test_rows_further_apart_than_the_kernels_reach(gpu):
	"""Column slices of a [tokens, batch, 3 d] buffer whose rows lie 3 * 2^20 elements apart, and single rows whose stride is as large."""
	from vit_amd import ops
	B, S, H, dh = 1 << 15, 3, 2, 16
	d = H * dh
	joint = torch.randn(S, B, 3 * d, device=gpu, generator=torch.Generator(device=gpu).manual_seed(30)).bfloat16().transpose(0, 1)
	parts = [joint[..., i * d:(i + 1) * d] for i in range(3)]
	leaves, dense = [t.detach().requires_grad_() for t in parts], [t.contiguous().requires_grad_() for t in parts]
	g = torch.randn(B, S, d, device=gpu).bfloat16()
	a, b = ops.biased_attention(*leaves, H, causal=True), ops.biased_attention(*dense, H, causal=True)
	assert torch.equal(a, b)
	for x, y in zip(torch.autograd.grad(a, leaves, g.transpose(0, 1).contiguous().transpose(0, 1)), torch.autograd.grad(b, dense, g)):
		assert torch.equal(x, y)
	with torch.no_grad():
		one = ops.biased_attention(parts[0][:, 1:2], parts[1][:, 2:], parts[2][:, 2:], H)
	assert torch.equal(one, parts[2][:, 2:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["shared", "per_image", "far", "with_lookup"])
def test_slopes_over_given_positions(gpu, dtype, kind):
	"""Distance slopes without a table over positions that are not the token indices: shared ones that repeat, each image's own, some 2^28 apart (a weight of 0
	there), and those of buckets that have a lookup too."""
	from vit_amd import ops
	B, H, Sq, Skv, dh = 2, 2, 70, 150, 40
	g_ = torch.Generator().manual_seed(31)
	q, k, v, g = make(B, H, H, Sq, Skv, dh, dtype, seed=32)
	shape = (B,) if kind == "per_image" else ()
	qp, kp = (torch.randint(-40, 40, (*shape, S), generator=g_).to(torch.int32) for S in (Sq, Skv))
	if kind == "far":
		qp[::7] += 1 << 28
		kp[::3] += 1 << 28
		kp[1::9] -= 1 << 28
	slopes = torch.tensor([0.5, 0.03125])
	leaves = [t.to(gpu).requires_grad_() for t in (q, k, v)]
	lookup = torch.zeros(3, dtype=torch.int32, device=gpu) if kind == "with_lookup" else None
	out = ops.biased_attention(*leaves, H, slopes=slopes.to(gpu), buckets=ops.RelativeBuckets(lookup, q_pos=qp.to(gpu), k_pos=kp.to(gpu)))
	got = dict(zip(["out", "dq", "dk", "dv"], [out.detach(), *torch.autograd.grad(out, leaves, g.to(gpu))]))
	check(got, *reference(q, k, v, g, H, H, slopes=slopes, q_pos=qp, k_pos=kp))


def test_buckets_without_a_table_or_slopes_are_refused(gpu):
	from vit_amd import ops
	x, p = torch.zeros(1, 4, 16, device=gpu), torch.zeros(4, dtype=torch.int32, device=gpu)
	with pytest.raises(ValueError, match="needed"):
		ops.RelativeBuckets(None)
	for kw in (dict(), dict(table=torch.zeros(3, 2, device=gpu))):
		with pytest.raises(ValueError, match="belong|lookup"):
			ops.biased_attention(x, x, x, 2, buckets=ops.RelativeBuckets(None, q_pos=p, k_pos=p), **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [0.0, 3.0])
@pytest.mark.parametrize("bias", ["none", "table", "slopes"])
@pytest.mark.parametrize("Sq,Skv", [(150, 150), (20, 900)])
def test_rows_that_meet_nobody_may_hold_anything(gpu, dtype, softcap, bias, Sq, Skv):
	"""Queries of a segment that no key has, and keys of one that no query has (neither is padding), hold NaN: zero gradients there, the others' as ever."""
	from vit_amd import ops
	H, dh = 2, 40
	q, k, v, g = make(2, H, H, Sq, Skv, dh, dtype, seed=33, gain=3.0 if softcap else 1.0)
	qs, ks = ((torch.arange(S) * 3 // S).to(torch.int32).repeat(2, 1) for S in (Sq, Skv))
	qs[:, 3::11], ks[:, 5::13] = 7, 1 + 8 * (torch.arange(5, Skv, 13) % 2).to(torch.int32)
	alone = ks == 9
	q[qs == 7], g[qs == 7], k[alone], v[alone] = (float("nan"),) * 4
	kw = dict(segments=(qs, ks), softcap=softcap)
	if bias == "table":
		pl = ops.RelativeBuckets.log_distance(16, 40, "cpu")
		kw.update(table=torch.randn(16, H, generator=torch.Generator().manual_seed(2)), lookup=pl.lookup, lo=pl.lo)
	elif bias == "slopes":
		kw["slopes"] = torch.tensor([0.5, 0.01])
	got = run(gpu, q, k, v, g, H, H, **kw)
	check(got, *reference(q, k, v, g, H, H, **kw))
	assert float(got["dq"][(qs == 7).to(gpu)].abs().max()) == 0.0 and float(got["dk"][alone.to(gpu)].abs().max()) == 0.0


def natural(q, k, v, dout, H, vis, softcap):
	"""out, dq, dk, dv in float64 with every hidden pair left out of each sum, as the definition has it: infinities and NaN go where the visible pairs take them."""
	B, Sq, _ = q.shape
	Skv, dh = k.shape[1], q.shape[2] // H
	heads = lambda t: t.double().view(B, -1, H, dh).transpose(1, 2)
	Q, K, V, G = (heads(t) for t in (q, k, v, dout))
	vis = vis[:, None]
	pairs = lambda a, b: (a[:, :, :, None, :] * b[:, :, None, :, :]).sum(-1)  # (no product that sums over rows)
	s = pairs(Q, K) * dh ** -0.5
	t = torch.tanh(s / softcap) if softcap else torch.zeros_like(s)
	p = torch.where(vis, torch.softmax(torch.where(vis, softcap * t if softcap else s, -math.inf), -1), 0.0)
	over = lambda w, x, m: torch.where(m[..., None], w[..., None] * x[:, :, None, :, :], 0.0).sum(3)
	out = over(p, V, vis)
	ds = p * (pairs(G, V) - (G * out).sum(-1, keepdim=True)) * (1 - t * t) * dh ** -0.5
	back = lambda w, x: over(w.transpose(2, 3), x, vis.transpose(2, 3))
	merge = lambda x: x.transpose(1, 2).reshape(B, -1, H * dh)
	return dict(out=merge(out), dq=merge(over(ds, K, vis)), dk=merge(back(ds, Q)), dv=merge(back(p, G)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mask", ["segments", "causal"])
@pytest.mark.parametrize("softcap", [0.0, 3.0])
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_specials_in_visible_places(gpu, dtype, mask, softcap, where, value):
	"""An infinity or a NaN in one column of two rows.  Results of rows that do not see one, and gradients of what only such rows see, keep their values; of
	the others everything that the definition makes an infinity or a NaN is one (a whole row may be, where the definition has one column)."""
	B, H, S, dh = 1, 2, 200, 40
	xs = dict(zip(("q", "k", "v", "dout"), make(B, H, H, S, S, dh, dtype, seed=34, gain=3.0 if softcap else 1.0)))
	seg = (torch.arange(S) // 50).to(torch.int32)[None]
	kw = dict(segments=(seg, seg)) if mask == "segments" else dict(causal=True)
	vis = visible(B, S, S, **kw)
	val, tol = reference(*xs.values(), H, H, softcap=softcap, **kw)
	rows = torch.zeros(S, dtype=torch.bool)
	rows[[70, 130]] = True  # (documents 1 and 2; the causal mask's queries from 70 on)
	xs[where][0, rows, 3] = value
	want = natural(*xs.values(), H, vis, softcap)
	got = run(gpu, *xs.values(), H, H, softcap=softcap, **kw)
	reached = dict(q=rows, dout=torch.zeros_like(rows)).get(where, (vis[0] & rows).any(1))  # queries whose out is
	back = rows if where == "dout" else reached  # queries whose gradients are
	keys = (vis[0] & back[:, None]).any(0)
	for n, touched in (("out", reached), ("dq", back), ("dk", keys), ("dv", keys)):
		a, w = got[n].double().cpu(), want[n]
		assert torch.isfinite(a[:, ~touched]).all() and ((a - val[n]).abs() <= tol[n] + 1e-12)[:, ~touched].all(), n
		assert not (torch.isfinite(a) & ~torch.isfinite(w)).any(), n
	assert 0 < int(back.sum()) < S


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_table_gradient_has_the_type_of_the_table(gpu, dtype):
	from vit_amd import ops
	q, k, v, g = (t.to(gpu) for t in make(2, 2, 2, 49, 49, 32, torch.bfloat16, seed=35))
	pl = ops.RelativeBuckets.grid(7, 7, gpu)
	table = torch.randn(169, 2, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)).half()
	grad = lambda t: torch.autograd.grad(ops.biased_attention(q, k, v, 2, table=t, buckets=pl), t, g)[0]
	want = grad(table.float().to(dtype).float().requires_grad_())
	got = grad(table.to(dtype).requires_grad_())
	assert got.dtype == dtype and torch.equal(got, want.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["causal", "segments", "slopes", "long", "all keys"])
def test_scores_that_are_all_minus_infinity_are_no_softmax(gpu, dtype, kind):
	"""An infinity in a query, or in every key, whose scores are -inf one and all: NaN, as the softmax of such a row is, while a query that sees no key is 0."""
	B, H, dh = 2, 2, 24
	Sq, Skv = dict(long=(3, 1500)).get(kind, (128, 128))
	q, k, v, g = make(B, H, H, Sq, Skv, dh, dtype, seed=36)
	k[..., 3] = -k[..., 3].abs() - 0.1  # (column 3 of head 0)
	kw, extra = {}, {}
	if kind in ("causal", "slopes"):
		kw = dict(causal=True)
	if kind == "slopes":
		extra = dict(slopes=torch.tensor([0.5, 0.25]))
	if kind == "segments":
		qs = (torch.arange(Sq) // 3).to(torch.int32).repeat(B, 1)
		ks = qs.clone()
		ks[:, 30:33] = 1000  # queries 30 .. 32 see nothing
		kw = dict(segments=(qs, ks))
	rows = torch.zeros(B, Sq, dtype=torch.bool)
	if kind == "all keys":
		k[..., 3] = -math.inf
		q[..., 3] = torch.where(torch.arange(Sq) % 2 == 0, q[..., 3].abs() + 0.1, q[..., 3])
	else:
		rows[:, [0, 2, 31] if Sq > 31 else [0, 2]] = True
		q[..., 3][rows] = math.inf
	got = run(gpu, q, k, v, g, H, H, **kw, **extra)
	want = natural(q, k, v, g, H, visible(B, Sq, Skv, **kw), 0.0)  # (slopes do not change what is finite)
	out, w = got["out"].double().cpu(), want["out"]
	if kind == "segments":
		assert float(out[:, 30:33].abs().max()) == 0.0 and bool(torch.isnan(out[:, [0, 2], :dh]).all())
		w[:, 30:33] = 0.0  # (the softmax of nothing, here 0)
	assert torch.equal(torch.isnan(out), torch.isnan(w))
	for n in ("dq", "dk", "dv"):
		a, x = got[n].double().cpu(), want[n]
		if kind != "segments":
			assert not (torch.isfinite(a) & ~torch.isfinite(x)).any(), n


@pytest.mark.parametrize("S,Skv,dh,H,Hkv", [(3, 3, 32, 1, 1), (8, 8, 80, 2, 1), (60, 60, 64, 4, 2), (1, 2, 128, 3, 3), (5, 900, 64, 2, 1), (40, 40, 7, 2, 2), (33, 70, 12, 2, 2), (300, 300, 20, 1, 1)])
@pytest.mark.parametrize("mask", ["causal", "documents", "none"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("bias", [False, True])
def test_score_gradients_where_weights_are_near_one(gpu, S, Skv, dh, H, Hkv, mask, softcap, bias):
	"""Large scores put most of a row's weight on one key, and dz = p (dp - delta) is a small difference there: delta = rowsum(dout o out) of a rounded out
	(an error of 2^-8 |out| |dout|) would be as far off as dz is large.  With what the rounding took, what is left of delta's error is that of the
	weights in out, rounded once each (u of them), but for the greatest, which is 1; rests below 2^-14 of out, which are not kept (3 F), and the float32
	sums (F).  Then one rounding of dz and one of the result."""
	from vit_amd import ops
	B = 4
	q, k, v, g = make(B, H, Hkv, S, Skv, dh, torch.bfloat16, seed=S + dh, gain=4.0)
	kw = dict(softcap=softcap)
	if mask == "causal":
		kw["causal"] = True
	if mask == "documents":
		kw["segments"] = tuple((torch.arange(n) // 3).to(torch.int32).repeat(B, 1) for n in (S, Skv))
	if bias:
		pl = ops.RelativeBuckets.log_distance(16, 40, "cpu")
		kw.update(table=torch.randn(16, H, generator=torch.Generator().manual_seed(3)), lookup=pl.lookup, lo=pl.lo)
	got = run(gpu, q, k, v, g, H, Hkv, **kw)
	val, fine = reference(*(t.float() for t in (q, k, v, g)), H, Hkv, **kw)  # (the bounds of float32 operands: neither rounding nor a rounded out in them)
	u, rounded = U[torch.bfloat16], rounded_scores(q, k, v, g, H, Hkv, **kw)
	for n in ("dq", "dk"):
		tol = 4 * fine[n] + rounded[n] + u * val[n].abs()
		a = got[n].double().cpu()
		worst = ((a - val[n]).abs() / (tol + 1e-12)).max().item()
		assert worst <= 1.0, f"{n}: {worst:.2f} times the bound"


def rounded_scores(q, k, v, dout, H, Hkv, softcap=0.0, table=None, lookup=None, lo=0, **mask):
	"""What one rounding of dz, and of every weight but a row's greatest in delta, can make of dq and dk, in float64."""
	B, Sq, _ = q.shape
	Skv, dh, u = k.shape[1], q.shape[2] // H, U[torch.bfloat16]
	heads = lambda t, n: t.double().view(B, -1, n, dh).transpose(1, 2)
	Q, G = heads(q, H), heads(dout, H)
	K, V = (heads(t, Hkv).repeat_interleave(H // Hkv, 1) for t in (k, v))
	s = Q @ K.transpose(2, 3) * dh ** -0.5
	t = torch.tanh(s / softcap) if softcap else torch.zeros_like(s)
	z = softcap * t if softcap else s
	if table is not None:
		d = torch.arange(Skv)[None] - torch.arange(Sq)[:, None] - (Skv - Sq)
		z = z + table.double()[lookup.long()[(d - lo).clamp(0, lookup.numel() - 1)]].permute(2, 0, 1)
	vis = visible(B, Sq, Skv, **mask)[:, None]
	p = torch.where(vis.any(-1, keepdim=True), torch.softmax(torch.where(vis, z, -1e30), -1), 0.0) * vis
	dp = G @ V.transpose(2, 3)
	others = torch.where(p == p.amax(-1, keepdim=True), 0.0, p)
	e = p * ((dp - (p * dp).sum(-1, keepdim=True)).abs() + (others * dp.abs()).sum(-1, keepdim=True)) * u * (1 - t * t) * dh ** -0.5
	merge = lambda x: x.transpose(1, 2).reshape(B, -1, x.shape[1] * dh)
	return dict(dq=merge(e @ K.abs()), dk=merge((e.transpose(2, 3) @ Q.abs()).view(B, Hkv, H // Hkv, Skv, dh).sum(2)))


@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("Skv", [700, 9000])
def test_weights_of_far_keys_sum_to_one_in_the_backward(gpu, softcap, Skv):
	"""One query whose visible keys lie thousands of positions in front of it, slopes of 0.8 and 0.3, float32: scores of thousands, a step of which is 2e-4 to
	5e-4.  The backward forms the same scores as the forward and divides by the same normaliser, so the weights of a row sum to one within the sums' F, and
	with them dv to dout: a normaliser that were rounded like a score would be off by half a step."""
	from vit_amd import ops
	B, H, dh = 16, 2, 16
	q, k, v, g = make(B, H, H, 1, Skv, dh, torch.float32, seed=37, gain=3.0 if softcap else 1.0)
	n = torch.randint(Skv // 4, Skv // 2, (B, 1), generator=torch.Generator().manual_seed(38))
	seg = torch.where(torch.arange(Skv) < n, 0, -1).to(torch.int32).to(gpu)
	leaves = [t.to(gpu).requires_grad_() for t in (q, k, v)]
	out = ops.biased_attention(*leaves, H, slopes=torch.tensor([0.8, 0.3], device=gpu), segments=(torch.zeros(B, 1, dtype=torch.int32, device=gpu), seg), softcap=softcap)
	dv = torch.autograd.grad(out, leaves, g.to(gpu))[2].double().cpu().sum(1, keepdim=True)
	assert float(((dv - g.double()).abs() / g.double().abs()).max()) <= F
