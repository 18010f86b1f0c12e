"""GPU: group normalisation with an activation over channels-last activations (ops.group_norm_act) against its definition in float64.

Tolerances: float32 statistics and sums carry relative errors of a few 2^-24 (a hundred terms at most are added one by one, the rest in trees): 2e-6 of the sum of
the terms' absolute values, and as much of every later quantity; a bfloat16 result is rounded once (half a step, 2^-8 of it).  dx is a difference that
cancels: its error is 4e-6 of the absolute values that go into it.  GELU's normal distribution function is good to 1.5e-7 absolute, its derivative likewise,
which 2e-6 covers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F = 4e-6
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16]


def act_of(z, act):
	if act == "silu":
		s = torch.sigmoid(z)
		return z * s, s * (1 + z * (1 - s))
	if act == "gelu":
		c = 0.5 * torch.erfc(-z / math.sqrt(2))
		return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
	if act == "relu":
		return z.clamp(min=0), (z > 0).double()
	if act == "relu6":
		return z.clamp(0, 6), ((z > 0) & (z < 6)).double()
	return z, torch.ones_like(z)


def reference(x, w, b, dy, groups, eps, act):
	B, C = x.shape[0], x.shape[-1]
	u = U[x.dtype]
	shape = (B, -1, groups, C // groups)
	x, dy = x.double().reshape(shape), dy.double().reshape(shape)
	w = (w.double() if w is not None else torch.ones(C, dtype=torch.float64)).reshape(groups, -1)
	b = (b.double() if b is not None else torch.zeros(C, dtype=torch.float64)).reshape(groups, -1)
	mean = x.mean((1, 3), keepdim=True)
	rstd = (x.var((1, 3), unbiased=False, keepdim=True) + eps).rsqrt()
	# the inputs' own size enters (x - mean): a mean far larger than the deviation costs its rounding
	err = F * (1 + x.abs().amax((1, 3), keepdim=True) * rstd * 2.0 ** -24 / F)
	xh = (x - mean) * rstd
	z = xh * w + b
	y, sl = act_of(z, act)
	val, tol = {}, {}
	val["y"], tol["y"] = y, u * y.abs() + err * (1 + (xh * w).abs() + b.abs()) * 2
	dz = dy * sl
	edz = err * dy.abs() * (1 + z.abs())
	val["dweight"], tol["dweight"] = (dz * xh).sum((0, 1)).reshape(C), (edz * (1 + xh.abs()) + err * (dz * xh).abs()).sum((0, 1)).reshape(C)
	val["dbias"], tol["dbias"] = dz.sum((0, 1)).reshape(C), (edz + err * dz.abs()).sum((0, 1)).reshape(C)
	h = dz * w
	m1, m2 = h.mean((1, 3), keepdim=True), (h * xh).mean((1, 3), keepdim=True)
	a1, a2 = h.abs().mean((1, 3), keepdim=True), (h * xh).abs().mean((1, 3), keepdim=True)
	eh = edz * w.abs()
	val["dx"] = rstd * (h - m1 - xh * m2)
	tol["dx"] = u * val["dx"].abs() + rstd * (eh + eh.mean((1, 3), keepdim=True) + (eh * xh.abs()).mean((1, 3), keepdim=True) * xh.abs() + err * (h.abs() + a1 + xh.abs() * a2 + a2))
	return val, tol


def check(got, val, tol):
	for n, x in got.items():
		a = x.double().cpu()
		b, t = val[n].reshape(a.shape), tol[n].reshape(a.shape)
		assert torch.isfinite(a).all(), n
		worst = ((a - b).abs() / (t + 1e-30)).max().item()
		assert worst <= 1.0, f"{n}: {worst:.2f} times the bound"


def run(gpu, x, w, b, dy, groups, eps, act):
	from vit_amd import ops
	xs = [t.to(gpu).requires_grad_() if t is not None else None for t in (x, w, b)]
	y = ops.group_norm_act(*xs, groups, eps=eps, act=act)
	have = [t for t in xs if t is not None]
	names = [n for n, t in zip(("dx", "dweight", "dbias"), xs) if t is not None]
	return dict({"y": y.detach()}, **dict(zip(names, torch.autograd.grad(y, have, dy.to(gpu)))))


def make(B, S, C, dtype, seed=0, mean=0.5):
	g = torch.Generator().manual_seed(seed)
	x = (torch.randn(B, S, C, generator=g) + mean * torch.randn(C, generator=g)).to(dtype)
	return x, 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g), torch.randn(B, S, C, generator=g).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,S,C,G", [(2, 49, 384, 32), (1, 1, 64, 4), (3, 165, 90, 6), (2, 50, 27, 9), (2, 784, 192, 32), (2, 3136, 96, 8), (1, 12544, 64, 32), (3, 5000, 36, 3), (2, 300, 1040, 16),
	(1, 700, 2080, 32), (2, 17, 4096, 1), (9, 5, 8, 8), (300, 7, 16, 2), (1, 40000, 8, 1), (17, 130, 24, 1)])
def test_shapes(gpu, dtype, B, S, C, G):
	"""Both forms (held in registers; two passes over slabs), channel counts that no vector load fits, groups that a vector straddles, groups of one channel
	and of all, batches beyond one run of the parameter sums."""
	t = make(B, S, C, dtype, seed=S + C)
	check(run(gpu, *t, G, 1e-5, "silu"), *reference(*t, G, 1e-5, "silu"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "relu", "relu6"])
@pytest.mark.parametrize("S", [60, 6000])
def test_activations(gpu, dtype, act, S):
	x, w, b, dy = make(2, S, 40, dtype, seed=S)
	if act == "relu6":
		w = 4 * w
	val, tol = reference(x, w, b, dy, 5, 1e-5, act)
	got = run(gpu, x, w, b, dy, 5, 1e-5, act)
	if act in ("relu", "relu6"):
		# within an error of a corner the derivative may be either side's: no input of these lies there
		x4 = x.double().reshape(2, S, 5, 8)
		z = (x4 - x4.mean((1, 3), keepdim=True)) * (x4.var((1, 3), unbiased=False, keepdim=True) + 1e-5).rsqrt() * w.double().reshape(5, 8) + b.double().reshape(5, 8)
		assert float(torch.minimum(z.abs(), (z - 6).abs()).min()) > 1e-6
	check(got, val, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("S", [30, 9000])
@pytest.mark.parametrize("have", ["weight", "bias", "neither"])
def test_without_parameters(gpu, dtype, S, have):
	x, w, b, dy = make(2, S, 24, dtype, seed=1)
	w, b = w if have == "weight" else None, b if have == "bias" else None
	val, tol = reference(x, w, b, dy, 4, 1e-3, "silu")
	check(run(gpu, x, w, b, dy, 4, 1e-3, "silu"), val, tol)


@pytest.mark.parametrize("S", [60, 7000])
def test_mean_far_larger_than_the_deviation(gpu, S):
	"""Mean 1000, deviation 1: a sum of squares about zero would lose the variance altogether (its rounding is 1000^2 * 2^-24 = 0.06)."""
	g = torch.Generator().manual_seed(2)
	x = 1000 + torch.randn(2, S, 32, generator=g)
	x[:, 0] = 0.0  # the first row, which serves as the shift of the sums, is an outlier
	w, b, dy = torch.ones(32), torch.zeros(32), torch.randn(2, S, 32, generator=g)
	check(run(gpu, x, w, b, dy, 4, 1e-5, "none"), *reference(x, w, b, dy, 4, 1e-5, "none"))


def test_constant_group_and_group_of_one(gpu):
	"""Variance zero: y = act(bias), and the gradient of a group of a single value is zero exactly."""
	from vit_amd import ops
	b = torch.randn(8, device=gpu)
	y = ops.group_norm_act(torch.full((2, 5, 8), 3.25, device=gpu), None, b, 2, act="silu")
	assert torch.allclose(y, torch.nn.functional.silu(b).expand(2, 5, 8), atol=1e-6)
	x, w = torch.randn(3, 1, 8, device=gpu, requires_grad=True), torch.randn(8, device=gpu)
	(dx,) = torch.autograd.grad(ops.group_norm_act(x, w, b, 8, act="gelu"), x, torch.randn(3, 1, 8, device=gpu))
	assert float(dx.abs().max()) == 0.0


def test_images_are_independent(gpu):
	"""An image that holds a NaN, or infinities, leaves the others' results and gradients as they are."""
	for S in (50, 8000):
		x, w, b, dy = (t.to(gpu) for t in make(3, S, 32, torch.bfloat16, seed=3))
		clean = run(gpu, x.cpu(), w.cpu(), b.cpu(), dy.cpu(), 4, 1e-5, "silu")
		x[1, 7, 3], x[1, 2] = float("nan"), float("inf")
		got = run(gpu, x.cpu(), w.cpu(), b.cpu(), dy.cpu(), 4, 1e-5, "silu")
		for i in (0, 2):
			assert torch.equal(got["y"][i], clean["y"][i]) and torch.equal(got["dx"][i], clean["dx"][i])


def test_layouts_streams_and_repeats(gpu):
	"""A transposed (NCHW) view, an unaligned buffer, four dimensions; the same bits every time and on another stream."""
	from vit_amd import ops
	x, w, b, dy = make(2, 36, 48, torch.bfloat16, seed=4)
	val, tol = reference(x, w, b, dy, 6, 1e-5, "gelu")
	wd, bd = w.to(gpu), b.to(gpu)
	nchw = x.transpose(1, 2).contiguous().to(gpu)
	f = lambda t: ops.group_norm_act(t, wd, bd, 6, act="gelu")
	check({"y": f(nchw.transpose(1, 2))}, val, tol)
	odd = torch.empty(2 * 36 * 48 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(2, 36, 48)
	odd.copy_(x)
	check({"y": f(odd)}, val, tol)
	four = f(x.to(gpu).view(2, 6, 6, 48))
	assert four.shape == (2, 6, 6, 48)
	check({"y": four}, val, tol)
	for S, C in ((784, 96), (9000, 96)):
		t = make(3, S, C, torch.bfloat16, seed=5)
		first = run(gpu, *t, 8, 1e-5, "silu")
		s = torch.cuda.Stream()
		for i in range(2):
			with torch.cuda.stream(s if i else torch.cuda.current_stream()):
				again = run(gpu, *t, 8, 1e-5, "silu")
			torch.cuda.synchronize()
			assert all(torch.equal(first[n], again[n]) for n in first)


@pytest.mark.parametrize("S", [196, 9000])
def test_captured_step_replays(gpu, S):
	from vit_amd import ops
	sets = [[t.to(gpu) for t in make(2, S, 64, torch.bfloat16, seed=30 + i)] for i in range(3)]

	def step(x, w, b, dy):
		y = ops.group_norm_act(x, w, b, 8, act="silu")
		return [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]

	eager = [step(*(t.clone().requires_grad_() for t in s[:3]), s[3]) for s in sets]
	static = [t.clone().requires_grad_() for t in sets[0][:3]] + [sets[0][3].clone()]
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
	for i in (0, 1, 2, 0):
		with torch.no_grad():
			for dst, src in zip(static, sets[i]):
				dst.copy_(src)
		graph.replay()
		torch.cuda.synchronize()
		for a, b in zip(res, eager[i]):
			assert torch.equal(a, b), i
		torch.randn(1000, device=gpu).sum().item()


@pytest.mark.parametrize("shape", [(0, 4, 8), (2, 0, 8)])
def test_nothing_to_normalise(gpu, shape):
	from vit_amd import ops
	x, w = torch.randn(shape, device=gpu, requires_grad=True), torch.ones(8, device=gpu, requires_grad=True)
	y = ops.group_norm_act(x, w, None, 2, act="silu")
	assert y.shape == x.shape
	dx, dw = torch.autograd.grad(y.sum(), (x, w))
	assert dx.shape == x.shape and float(dw.abs().sum()) == 0.0


def test_gradient_sinks(gpu):
	from vit_amd import ops
	x, w, b, dy = (t.to(gpu) for t in make(2, 100, 32, torch.bfloat16, seed=6))
	w, b = torch.nn.Parameter(w), torch.nn.Parameter(b)
	f = lambda: ops.group_norm_act(x.requires_grad_(), w, b, 4, act="silu")
	dw, db = torch.autograd.grad(f(), (w, b), dy)
	bw, bb = torch.ones_like(w), torch.ones_like(b)
	for both in (True, False):
		bw.fill_(1.0)
		bb.fill_(1.0)
		w.grad = b.grad = None
		ops.register_grad_sink(w, bw)
		if both:
			ops.register_grad_sink(b, bb)
		try:
			f().backward(dy)
		finally:
			ops.unregister_grad_sink(w)
			ops.unregister_grad_sink(b)
		assert w.grad is None and torch.equal(bw, dw + 1.0)
		assert (b.grad is None and torch.equal(bb, db + 1.0)) if both else torch.equal(b.grad, db)


def test_gradient_against_differences(gpu):
	"""Central differences along random directions, h = 2^-6: the curvature term is O(h^2) of a smooth function of unit size, the rounding term
	2^-24 / h; 1 % covers both."""
	from vit_amd import ops
	g = torch.Generator().manual_seed(8)
	xs = [t.to(gpu) for t in make(2, 30, 12, torch.float32, seed=7)]
	dy = xs.pop()
	f = lambda x, w, b: ops.group_norm_act(x, w, b, 3, act="gelu")
	leaves = [t.clone().requires_grad_() for t in xs]
	grads = torch.autograd.grad(f(*leaves), leaves, dy)
	for n in range(3):
		e, h = torch.randn(xs[n].shape, generator=g).to(gpu), 2.0 ** -6
		with torch.no_grad():
			at = lambda s: (f(*[x + s * h * e if i == n else x for i, x in enumerate(xs)]).double() * dy.double()).sum()
			num = float((at(1) - at(-1)) / (2 * h))
		ana = float((grads[n].double() * e.double()).sum())
		assert abs(num - ana) < 1e-2 * max(abs(num), float(grads[n].double().norm()))


@pytest.mark.parametrize("act", ["none", "relu", "relu6", "silu", "gelu"])
@pytest.mark.parametrize("S", [10, 4000])
def test_a_nan_stays_in_its_group(gpu, act, S):
	"""One NaN makes its image's group NaN, through every activation, and leaves the others' bits alone."""
	from vit_amd import ops
	x, w, b, dy = (t.to(gpu) for t in make(2, S, 32, torch.bfloat16, seed=21))
	f = lambda t: ops.group_norm_act(t, w, b, 4, act=act)
	want = f(x)
	bad = x.clone()
	bad[1, 3, 9] = float("nan")
	got = f(bad)
	assert bool(got[1, :, 8:16].isnan().all())
	got[1, :, 8:16] = want[1, :, 8:16]
	assert torch.equal(got, want)


def test_a_weight_of_another_type_is_read_at_each_replay(gpu):
	from vit_amd import ops
	x, w, b, _ = (t.to(gpu) for t in make(2, 30, 32, torch.bfloat16, seed=22))
	w = w.bfloat16()
	f = lambda: ops.group_norm_act(x, w, b, 4, act="silu")
	f()
	side = torch.cuda.Stream()
	side.wait_stream(torch.cuda.current_stream())
	with torch.cuda.stream(side):
		f()
	torch.cuda.current_stream().wait_stream(side)
	graph = torch.cuda.CUDAGraph()
	with torch.cuda.graph(graph):
		y = f()
	for i in range(3):
		w.copy_(torch.randn(32, device=gpu))
		graph.replay()
		torch.cuda.synchronize()
		assert torch.equal(y, f()), i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,G", [(96, 32), (384, 32), (768, 32), (72, 9), (90, 6)])
@pytest.mark.parametrize("S", [1, 2, 4, 7])
def test_few_positions(gpu, dtype, S, C, G):
	"""Images of fewer positions than a vector has values, whose last slice of channels is narrower than the others: more channels than threads with rows."""
	t = make(3, S, C, dtype, seed=S + C)
	check(run(gpu, *t, G, 1e-5, "silu"), *reference(*t, G, 1e-5, "silu"))


def test_gelu_in_float32_keeps_its_digits(gpu):
	"""Values +-1 in equal numbers and eps 0: mean 0, deviation 1, so that z is the weight, +-, without an error.  y = z Phi(z): Phi's argument z / sqrt 2 carries
	two roundings (2^-23 together), which exp(-z^2 / 2) turns into z^2 as much where it decides (z < 0), and erfc and three products a few units in the last place
	more: (z^2 + 8) 2^-23.  The derivative is Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi), the exponential good to (z^2 + 4) 2^-23 of itself."""
	from vit_amd import ops
	C = 64
	w = torch.cat([torch.linspace(0.01, 6, C // 2 - 1), -torch.tensor([0.5, 1.0]), torch.linspace(0.02, 5, C // 2 - 1)])
	for S in (4, 6000):
		x = torch.ones(1, S, C)
		x[:, ::2] = -1
		xg, wg = x.to(gpu).requires_grad_(), w.to(gpu)
		y = ops.group_norm_act(xg, wg, None, 1, eps=0.0, act="gelu")
		z = x.double() * w.double()
		cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
		err = ((y.detach().double().cpu() - z * cdf).abs() / ((z * cdf).abs() * (z * z + 8) * 2.0 ** -23)).max()
		assert float(err) <= 1.0, (S, float(err))
		# dbias of one channel sums its slopes: channel by channel, through a gradient that is 1 in one row alone
		b = torch.zeros(C, device=gpu, requires_grad=True)
		for row in (0, 1):
			dy = torch.zeros(1, S, C, device=gpu)
			dy[:, row] = 1
			(db,) = torch.autograd.grad(ops.group_norm_act(xg.detach(), wg, b, 1, eps=0.0, act="gelu"), b, dy)
			zr, cr = z[0, row], cdf[0, row]
			bell = zr * torch.exp(-zr * zr / 2) / math.sqrt(2 * math.pi)
			tol = (cr * (zr * zr + 8) + bell.abs() * (zr * zr + 8)) * 2.0 ** -23
			assert float(((db.double().cpu() - cr - bell).abs() / tol).max()) <= 1.0, (S, row)


@pytest.mark.parametrize("S", [784, 20000])
@pytest.mark.parametrize("G", [1, 8, 32])
@pytest.mark.parametrize("rows", [(0,), (0, 9), (5,)])
def test_outlying_rows_cost_no_digits(gpu, S, G, rows):
	"""Rows a hundred deviations out, the first among them.  All terms of the squared deviations are positive: at most 48 roundings on a term's way through the
	sums (8 rows one by one, then runs and trees), and 24 more where a few rows' squares are taken about one of them, 2^-24 each: 72 in the variance, half of
	that in rstd, and 4 for its root and quotient.  One factor for a whole group: the ratio of y to its value, over all of the group."""
	g = torch.Generator().manual_seed(40)
	x = torch.randn(2, S, 64, generator=g)
	for r in rows:
		x[:, r] += 100.0 * torch.sign(torch.randn(2, 64, generator=g)) if r else 100.0
	from vit_amd import ops
	y = ops.group_norm_act(x.to(gpu), None, None, G, eps=0.0).double().cpu().reshape(2, S, G, -1)
	xd = x.double().reshape(2, S, G, -1)
	want = (xd - xd.mean((1, 3), keepdim=True)) * xd.var((1, 3), unbiased=False, keepdim=True).rsqrt()
	ratio = (y * want).sum((1, 3)) / want.square().sum((1, 3))
	assert float((ratio - 1).abs().max()) <= 40 * 2.0 ** -24, float((ratio - 1).abs().max() * 2 ** 24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_parameter_gradients_have_the_parameters_types(gpu, dtype):
	from vit_amd import ops
	x, w, b, dy = (t.to(gpu) for t in make(2, 50, 32, torch.bfloat16, seed=41))
	w, b = w.half(), b.half()
	grads = lambda *p: torch.autograd.grad(ops.group_norm_act(x, *p, 4, act="silu"), p, dy)
	want = grads(*(t.to(dtype).float().requires_grad_() for t in (w, b)))
	for g, r in zip(grads(*(t.to(dtype).requires_grad_() for t in (w, b))), want):
		assert g.dtype == dtype and torch.equal(g, r.to(dtype))
