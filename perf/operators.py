"""Cases for the attention with biased, capped and masked scores and for the channels-last group normalisation.

Attention.  q [B, Sq, H * dh], k and v [B, Skv, Hkv * dh]; query head h reads key head h // (H / Hkv):

    s = q k^T / sqrt(dh);  z = cap * tanh(s / cap) (or s);  z += table[bucket(kpos - qpos), h];  z -= slope[h] * |kpos - qpos|
    out = softmax over the visible keys (z) v;  a query that sees no key gives 0

bucket(d) = lookup[clamp(d - lo, 0, len(lookup) - 1)].  A key is visible when its segment number equals the query's and is not
negative, and, with `causal`, when its index is at most the query's (aligned at the end) or below the sequence's prefix length.
A training pass returns out and the gradients of q, k, v and table for a given gradient of out.

Group normalisation.  x [B, S, C] token-major; the C channels in G groups; y = act((x - mean) * rstd * gamma + beta) with
mean and variance over the S * C / G values of each image and group.  A training pass returns y and the gradients of x, gamma, beta.
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
	return [
		# relative-bias attention: third stage of the conv + attention hybrid at 224 x 224 (28 x 28 tokens, 32 heads of 12)
		dict(name="grid bias 28x28 d12 train", op="attn", B=16, gh=28, gw=28, H=32, Hkv=32, dh=12, dtype="bf16", bias="grid", train=True),
		# the 14 x 14 token grid of a 224 x 224 image at patch 16, 12 heads of 64
		dict(name="grid bias 14x14 d64 train", op="attn", B=64, gh=14, gw=14, H=12, Hkv=12, dh=64, dtype="bf16", bias="grid", train=True),
		# parity-style float32 training of a small odd grid
		dict(name="grid bias 9x13 f32 train", op="attn", B=2, gh=9, gw=13, H=3, Hkv=3, dh=40, dtype="f32", bias="grid", train=True),
		# one long token sequence with logarithmic distance buckets
		dict(name="log buckets 4096 train", op="attn", B=1, Sq=4096, Skv=4096, H=8, Hkv=8, dh=64, dtype="bf16", bias="log", train=True),
		# images of many resolutions packed into one row of 8192 patches, a padded tail behind the last one
		dict(name="documents 8192 train", op="attn", B=1, Sq=8192, Skv=8192, H=12, Hkv=12, dh=64, dtype="bf16", mask="documents", train=True),
		# image prefix seen both ways, text behind it causal, capped scores, four query heads to a key head
		dict(name="prefix cap d128 train", op="attn", B=2, Sq=2048, Skv=2048, H=16, Hkv=4, dh=128, dtype="bf16", mask="prefix", cap=30.0, train=True),
		# one class-token query over a long padded token set, distance bias: the single-token serving form
		dict(name="one query 16384 slopes", op="attn", B=16, Sq=1, Skv=16384, H=12, Hkv=12, dh=64, dtype="bf16", mask="padded", bias="slopes", train=False),
		# the smallest calls: a short float32 sequence, capped, forward only
		dict(name="short prefix cap f32", op="attn", B=2, Sq=65, Skv=65, H=3, Hkv=3, dh=64, dtype="f32", mask="prefix", cap=30.0, train=False),
		# group normalisation of a 7 x 7 map, forward only: latency
		dict(name="group norm 7x7 silu", op="gn", B=2, S=49, C=384, G=32, dtype="bf16", act="silu", train=False),
		# hidden layer of the hybrid's second conv stage behind its stride (28 x 28, 4 * 192 channels), batch 128
		dict(name="group norm 28x28 silu train", op="gn", B=128, S=784, C=768, G=32, dtype="bf16", act="silu", train=True),
		# hidden layer of the first conv stage (112 x 112, 4 * 64 channels)
		dict(name="group norm 112x112 silu train", op="gn", B=64, S=12544, C=256, G=32, dtype="bf16", act="silu", train=True),
		# odd sizes in float32, 15 channels a group
		dict(name="group norm 15x11 gelu f32 train", op="gn", B=3, S=165, C=90, G=6, dtype="f32", act="gelu", train=True),
	]


def _spread(rng, lo, hi):
	"""A whole number from lo to hi, even over its logarithm."""
	return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
	kind = rng.choice(["grid", "log", "documents", "prefix", "query", "gn", "gn"])
	dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
	train = rng.random() < 0.7
	if kind == "gn":
		G = rng.choice([1, 2, 4, 8, 16, 32])
		C = G * rng.choice([1, 2, 3, 4, 8, 12, 16, 24, 27]) if G < 32 else rng.choice([32, 64, 96, 192, 256, 384, 768])
		S, B = _spread(rng, 1, 12544), _spread(rng, 1, 128)
		while B > 1 and B * S * C > 100_000_000:
			B = (B + 1) // 2
		return dict(op="gn", B=B, S=S, C=C, G=G, dtype=dtype, act=rng.choice(["none", "silu", "gelu"]), train=train)
	Hkv = rng.choice([1, 2, 3, 4, 6, 8])
	H = Hkv * rng.choice([1, 1, 2, 4])
	dh = rng.choice([8, 12, 24, 32, 40, 64, 64, 80, 96, 128])
	c = dict(op="attn", H=H, Hkv=Hkv, dh=dh, dtype=dtype, train=train)
	most = 150_000_000 if dtype == "bf16" else 30_000_000  # scores of all heads
	if kind == "grid":
		gh, gw = rng.randint(1, 32), rng.randint(1, 32)
		B, n = _spread(rng, 1, 64), (gh * gw) ** 2
		c.update(gh=gh, gw=gw, bias="grid", cap=rng.choice([0.0, 0.0, 30.0]))
	elif kind == "query":
		S = _spread(rng, 16, 16384)
		B, Sq = _spread(rng, 1, 16), rng.choice([1, 1, 1, 2, 5, 16])
		n = 16 * S
		c.update(Sq=Sq, Skv=S, bias=rng.choice(["slopes", "log", "none"]), mask="padded", cap=rng.choice([0.0, 30.0]))
	else:
		S = _spread(rng, 1, 4096)
		Sq = S if rng.random() < 0.7 else _spread(rng, 1, S)
		B, n = _spread(rng, 1, 16), S * Sq
		c.update(Sq=Sq, Skv=S)
		if kind == "log":
			c.update(bias="log", mask=rng.choice(["none", "prefix"]))
		elif kind == "documents":
			c.update(Sq=S, mask="documents", cap=rng.choice([0.0, 30.0]), bias=rng.choice(["none", "slopes"]))
			n = S * S
		else:
			c.update(mask="prefix", cap=rng.choice([0.0, 30.0]), bias=rng.choice(["none", "slopes"]))
	while B > 1 and B * H * n > most:
		B = (B + 1) // 2
	while c["H"] > 1 and c["H"] * B * n > most:
		c["H"] = c["Hkv"] = max(1, c["H"] // 2)
	c["B"] = B
	return c


def _sizes(c):
	return (c["gh"] * c["gw"],) * 2 if "gh" in c else (c["Sq"], c["Skv"])


def log_buckets(n_bucket, max_distance):
	"""Bucket of every distance -max_distance .. max_distance: half of the buckets for keys behind the query, half for keys in front;
	in each half the first ones hold one distance, the others logarithmically growing ranges."""
	half, exact_ = n_bucket // 2, n_bucket // 4
	d = torch.arange(-max_distance, max_distance + 1)
	a = d.abs()
	far = exact_ + (torch.log(a.clamp(min=1).double() / exact_) / math.log(max_distance / exact_) * (half - exact_) + 1e-9).floor().long()
	return torch.where(a < exact_, a, far.clamp(max=half - 1)) + torch.where(d > 0, half, 0)


def prepare(case, seed):
	g = torch.Generator(device="cuda").manual_seed(seed)
	dt = DTYPES[case["dtype"]]
	rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
	c = dict(case)
	st = {"case": c}
	if c["op"] == "gn":
		B, S, C = c["B"], c["S"], c["C"]
		st["x"] = (rnd(B, S, C) + 0.5 * rnd(C)).to(dt)
		st["weight"], st["bias"] = 1 + 0.2 * rnd(C), 0.2 * rnd(C)
		st["dy"] = rnd(B, S, C).to(dt) if c["train"] else None
		return st
	B, H, Hkv, dh = c["B"], c["H"], c["Hkv"], c["dh"]
	Sq, Skv = _sizes(c)
	gain = 3.0 if c.get("cap") else 1.0  # capped scores are large ones
	st["q"] = (gain * rnd(B, Sq, H * dh)).to(dt)
	st["k"], st["v"] = rnd(B, Skv, Hkv * dh).to(dt), rnd(B, Skv, Hkv * dh).to(dt)
	st["dout"] = rnd(B, Sq, H * dh).to(dt) if c["train"] else None
	st.update(table=None, lookup=None, lo=0, qpos=None, kpos=None, slopes=None, qseg=None, kseg=None, prefix=None)
	bias, mask = c.get("bias", "none"), c.get("mask", "none")
	if bias == "grid":
		gh, gw = c["gh"], c["gw"]
		code = (torch.arange(gh)[:, None] * (2 * gw - 1) + torch.arange(gw)).reshape(-1)
		st["qpos"] = st["kpos"] = code.to(torch.int32).cuda()
		st["lookup"] = torch.arange((2 * gh - 1) * (2 * gw - 1), dtype=torch.int32).cuda()
		st["lo"] = -((gh - 1) * (2 * gw - 1) + gw - 1)
		st["table"] = 0.5 * rnd((2 * gh - 1) * (2 * gw - 1), H)
	elif bias == "log":
		st["lookup"], st["lo"] = log_buckets(32, 128).to(torch.int32).cuda(), -128
		st["table"] = 0.5 * rnd(32, H)
	elif bias == "slopes":
		st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)
	if mask == "documents":  # ragged pieces in a row, the last few tokens padding
		u = torch.rand(B, Skv, device="cuda", generator=g)
		seg = (u < 1.0 / max(2.0, min(400.0, Skv / 4))).cumsum(1).to(torch.int32)
		seg[:, Skv - Skv // 20:] = -1
		st["qseg"] = st["kseg"] = seg
	elif mask == "padded":  # sequences of different lengths behind one another in a batch
		n = torch.randint(max(1, Skv // 2), Skv + 1, (B, 1), device="cuda", generator=g)
		st["kseg"] = torch.where(torch.arange(Skv, device="cuda") < n, 0, -1).to(torch.int32)
		st["qseg"] = torch.zeros(B, Sq, dtype=torch.int32, device="cuda")
	elif mask == "prefix":
		st["prefix"] = torch.randint(0, Skv // 2 + 1, (B,), device="cuda", generator=g).to(torch.int32)
	return st


# ---- plain forms: float32 throughout, gradients by their formulas, rounded once ------------------------------------------------

def _distance(st, Sq, Skv, device):
	"""kpos - qpos [Sq, Skv]; without positions the index, queries aligned with the last keys."""
	qp = st["qpos"].long() if st["qpos"] is not None else torch.arange(Sq, device=device) + (Skv - Sq)
	kp = st["kpos"].long() if st["kpos"] is not None else torch.arange(Skv, device=device)
	return kp[None, :] - qp[:, None]


def _hidden(st, Sq, Skv, device):
	"""True where a key is not visible: [B, 1, Sq, Skv], or None."""
	hid = None
	if st["kseg"] is not None:
		hid = (st["qseg"][:, :, None] != st["kseg"][:, None, :]) | (st["kseg"][:, None, :] < 0)
	if st["prefix"] is not None:
		i, j = torch.arange(Sq, device=device)[:, None] + (Skv - Sq), torch.arange(Skv, device=device)[None, :]
		behind = (j > i)[None] & (j[None] >= st["prefix"].long()[:, None, None])
		hid = behind if hid is None else hid | behind
	return None if hid is None else hid[:, None]


def _attention_plain(st):
	c = st["case"]
	B, H, Hkv, dh, dt = c["B"], c["H"], c["Hkv"], c["dh"], DTYPES[c["dtype"]]
	Sq, Skv = _sizes(c)
	cap, dev = c.get("cap", 0.0), st["q"].device
	heads = lambda t, n: t.float().view(B, -1, n, dh).transpose(1, 2)  # noqa: E731
	q = heads(st["q"], H)
	k, v = (heads(st[n], Hkv).repeat_interleave(H // Hkv, 1) for n in ("k", "v"))
	scale = dh ** -0.5
	z = q @ k.transpose(2, 3) * scale
	t = None
	if cap:
		t = torch.tanh(z / cap)
		z = cap * t
	if st["table"] is not None:
		d = _distance(st, Sq, Skv, dev)
		at = (d - st["lo"]).clamp(0, st["lookup"].numel() - 1)
		z = z + st["table"].float().t()[:, st["lookup"].long()][:, at]
	if st["slopes"] is not None:
		z = z - st["slopes"].float()[:, None, None] * _distance(st, Sq, Skv, dev).abs().float()
	hid = _hidden(st, Sq, Skv, dev)
	if hid is not None:
		z = z.masked_fill(hid, -math.inf)
	m = z.amax(-1, keepdim=True)
	p = torch.exp(z - torch.where(m == -math.inf, 0.0, m))
	total = p.sum(-1, keepdim=True)
	p = p / torch.where(total == 0, 1.0, total)
	merge = lambda x, n: x.transpose(1, 2).reshape(B, -1, n * dh).to(dt)  # noqa: E731
	out = {"out": merge(p @ v, H)}
	if not c["train"]:
		return out
	do = heads(st["dout"], H)
	shared = lambda x: x.view(B, Hkv, H // Hkv, Skv, dh).sum(2)  # noqa: E731
	out["dv"] = merge(shared(p.transpose(2, 3) @ do), Hkv)
	dp = do @ v.transpose(2, 3)
	dz = p * (dp - (p * dp).sum(-1, keepdim=True))
	if st["table"] is not None:
		# many values to a bucket: brought into the buckets' order and summed in 64 bits, each bucket between its ends
		bucket = st["lookup"].long()[at].reshape(-1)
		order = torch.argsort(bucket)
		run_sum = F.pad(dz.sum(0, dtype=torch.float64).view(H, -1)[:, order].cumsum(1), (1, 0))
		ends = torch.searchsorted(bucket[order], torch.arange(st["table"].shape[0] + 1, device=dev))
		out["dtable"] = (run_sum[:, ends[1:]] - run_sum[:, ends[:-1]]).t().contiguous().float()
	if cap:
		dz = dz * (1 - t * t)
	dz = dz * scale
	out["dq"] = merge(dz @ k, H)
	out["dk"] = merge(shared(dz.transpose(2, 3) @ q), Hkv)
	return out


def _act_plain(z, act):
	"""act(z) and its derivative."""
	if act == "silu":
		s = torch.sigmoid(z)
		return z * s, s * (1 + z * (1 - s))
	if act == "gelu":
		cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
		return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
	return z, torch.ones_like(z)


def _group_norm_plain(st):
	c = st["case"]
	B, S, C, G, dt = c["B"], c["S"], c["C"], c["G"], DTYPES[c["dtype"]]
	x = st["x"].float().view(B, S, G, C // G)
	mean = x.mean((1, 3), keepdim=True)
	xc = x - mean
	rstd = torch.rsqrt((xc * xc).mean((1, 3), keepdim=True) + 1e-5)
	xhat = xc * rstd
	w, b = st["weight"].view(G, C // G), st["bias"].view(G, C // G)
	y, slope = _act_plain(xhat * w + b, c["act"])
	out = {"y": y.view(B, S, C).to(dt)}
	if not c["train"]:
		return out
	dz = st["dy"].float().view(B, S, G, C // G) * slope
	out["dweight"] = (dz * xhat).sum((0, 1), dtype=torch.float64).float().view(C)
	out["dbias"] = dz.sum((0, 1), dtype=torch.float64).float().view(C)
	dh = dz * w
	dx = rstd * (dh - dh.mean((1, 3), keepdim=True) - xhat * (dh * xhat).mean((1, 3), keepdim=True))
	out["dx"] = dx.view(B, S, C).to(dt)
	return out


def _attention_own(st):
	from vit_amd import ops
	c = st["case"]
	buckets = None
	if st["table"] is not None:
		buckets = ops.RelativeBuckets(st["lookup"], st["lo"], q_pos=st["qpos"], k_pos=st["kpos"])
	segments = (st["qseg"], st["kseg"]) if st["kseg"] is not None else None
	kw = dict(n_kv_head=c["Hkv"], softcap=c.get("cap", 0.0), buckets=buckets, slopes=st["slopes"], segments=segments,
		causal=st["prefix"] is not None, prefix=st["prefix"])
	if not c["train"]:
		with torch.no_grad():
			return {"out": ops.biased_attention(st["q"], st["k"], st["v"], c["H"], table=st["table"], **kw)}
	names = ["q", "k", "v"] + (["table"] if st["table"] is not None else [])
	leaves = {n: st[n].detach().requires_grad_() for n in names}
	out = ops.biased_attention(leaves["q"], leaves["k"], leaves["v"], c["H"], table=leaves.get("table"), **kw)
	grads = torch.autograd.grad(out, list(leaves.values()), st["dout"])
	return dict({"out": out.detach()}, **{"d" + n: t for n, t in zip(names, grads)})


def _group_norm_own(st):
	from vit_amd import ops
	c = st["case"]
	if not c["train"]:
		with torch.no_grad():
			return {"y": ops.group_norm_act(st["x"], st["weight"], st["bias"], c["G"], act=c["act"])}
	x, w, b = (st[n].detach().requires_grad_() for n in ("x", "weight", "bias"))
	y = ops.group_norm_act(x, w, b, c["G"], act=c["act"])
	dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"])
	return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def run(state):
	if state["case"]["op"] == "attn":
		return _attention_own(state) if own else _attention_plain(state)
	return _group_norm_own(state) if own else _group_norm_plain(state)


def work(case):
	c = case
	e = 2 if c["dtype"] == "bf16" else 4
	if c["op"] == "gn":
		n = c["B"] * c["S"] * c["C"]
		passes = 5 if c["train"] else 2  # x, y; dy, x, dx
		return {"bytes": n * e * passes + 16 * c["C"], "flops": n * (30 if c["train"] else 10)}
	B, H, Hkv, dh = c["B"], c["H"], c["Hkv"], c["dh"]
	Sq, Skv = _sizes(c)
	rows_q, rows_k = B * Sq * H * dh, B * Skv * Hkv * dh
	share = 1.0  # of the scores that are visible, on average
	if c.get("mask") == "prefix":
		share = 1.0 - 0.5 * Sq / Skv * 0.58  # causal, but for prefixes that are a quarter of the keys on average
	elif c.get("mask") == "documents":
		share = min(1.0, 2.0 * max(2.0, min(400.0, Skv / 4)) / Skv)
	elif c.get("mask") == "padded":
		share = 0.75
		rows_k = rows_k * share
	products = 7 if c["train"] else 2  # forward q k^T, p v; backward those scores again and four products
	return {"bytes": e * ((2 * rows_q + 2 * rows_k) + (2 * rows_q + rows_q + 4 * rows_k if c["train"] else 0)), "flops": products * 2.0 * B * H * Sq * Skv * dh * share}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------

def exact(case, seed):
	st = prepare(case, seed)
	c = st["case"]
	return _exact_group_norm(st, c) if c["op"] == "gn" else _exact_attention(st, c)


def _exact_group_norm(st, c):
	B, S, C, G = c["B"], c["S"], c["C"], c["G"]
	w, b = (st[n].double().requires_grad_() for n in ("weight", "bias"))
	ys, dxs = [], []
	for i in range(B):
		x = st["x"][i].double().requires_grad_()
		xg = x.t().reshape(G, -1)
		var, mean = torch.var_mean(xg, 1, unbiased=False, keepdim=True)
		z = ((xg - mean) / torch.sqrt(var + 1e-5)).reshape(C, S).t() * w + b
		y = z / (1 + torch.exp(-z)) if c["act"] == "silu" else 0.5 * z * torch.erfc(-z / math.sqrt(2)) if c["act"] == "gelu" else z
		ys.append(y.detach())
		if c["train"]:
			y.backward(st["dy"][i].double())
			dxs.append(x.grad)
	out = {"y": torch.stack(ys)}
	if c["train"]:
		out.update(dx=torch.stack(dxs), dweight=w.grad, dbias=b.grad)
	return out


def _exact_attention(st, c):
	B, H, Hkv, dh = c["B"], c["H"], c["Hkv"], c["dh"]
	Sq, Skv = _sizes(c)
	cap, train = c.get("cap", 0.0), c["train"]
	dev = st["q"].device
	table = st["table"].double().requires_grad_(train) if st["table"] is not None else None
	qi, kj = torch.arange(Skv - Sq, Skv, device=dev), torch.arange(Skv, device=dev)
	qp, kp = (st["qpos"], st["kpos"]) if st["qpos"] is not None else (qi, kj)
	diff = torch.sub(kp.long().unsqueeze(0), qp.long().unsqueeze(1))
	outs, grads = [], []
	dtable = torch.zeros_like(table) if table is not None else None
	for b in range(B):
		q, k, v = (st[n][b].double().requires_grad_(train) for n in ("q", "k", "v"))
		o = torch.zeros(Sq, H * dh, dtype=torch.float64, device=dev)
		parts = []
		for h in range(H):
			kv = h // (H // Hkv)
			s = torch.mm(q[:, h * dh:(h + 1) * dh], k[:, kv * dh:(kv + 1) * dh].t()) / math.sqrt(dh)
			if cap:
				e = torch.exp(-2 * s.abs() / cap)
				s = cap * torch.sign(s) * (1 - e) / (1 + e)
			if table is not None:
				per = table[:, h][st["lookup"].long()]
				s = s + per[torch.clamp(diff - st["lo"], 0, st["lookup"].numel() - 1)]
			if st["slopes"] is not None:
				s = s - st["slopes"][h].double() * diff.abs()
			seen = torch.ones(Sq, Skv, dtype=torch.bool, device=dev)
			if st["kseg"] is not None:
				seen &= torch.eq(st["qseg"][b].unsqueeze(1), st["kseg"][b].unsqueeze(0)) & (st["kseg"][b] >= 0)
			if st["prefix"] is not None:
				seen &= (kj <= qi.unsqueeze(1)) | (kj < st["prefix"][b])
			some = seen.any(1)
			w = torch.softmax(torch.where(seen, s, torch.full_like(s, -1e300)), 1) * (seen & some.unsqueeze(1))
			part = torch.mm(w, v[:, kv * dh:(kv + 1) * dh])
			o[:, h * dh:(h + 1) * dh] = part.detach()
			if train:
				part.backward(st["dout"][b, :, h * dh:(h + 1) * dh].double())
		outs.append(o)
		if train:
			grads.append((q.grad, k.grad, v.grad))
	out = {"out": torch.stack(outs)}
	if train:
		for n, parts in zip(("dq", "dk", "dv"), zip(*grads)):
			out[n] = torch.stack(parts)
		if table is not None:
			out["dtable"] = table.grad
	return out
