"""Shared-prefix attention in 64 bits, and how far a kernel that rounds where the documentation says may be from it."""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}          # half a step, relative
TOP = {"int8": 127.0, "e4m3": 448.0}
F32 = 2.0 ** -24


def randn(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale


def quantise(rows, fmt):
    """One scale a row, codes round(row * top / max|row|), in float32."""
    amax = rows.abs().amax(-1, keepdim=True)
    y = (rows * (torch.full_like(amax, TOP[fmt]) / amax)).clamp(-TOP[fmt], TOP[fmt])
    codes = torch.round(y).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    return codes, (amax / torch.full_like(amax, TOP[fmt])).squeeze(-1)


class Part:
    """Keys and values (..., keys, d): as 16-bit tensors, or as codes and scales, of rows of uneven size."""

    def __init__(self, shape, fmt, dtype, seed):
        self.fmt = fmt
        rows = [randn(shape, seed + i) * torch.exp(0.5 * randn(shape[:-1] + (1,), seed + 2 + i)) for i in range(2)]
        if fmt == "none":
            self.k, self.v = (t.to(dtype) for t in rows)
        else:
            (self.k, self.ks), (self.v, self.vs) = (quantise(t, fmt) for t in rows)

    def numbers(self, shifted=False):
        """(keys, values) in 64 bits.  shifted: every key with its neighbour's scale."""
        if self.fmt == "none":
            return self.k.double(), self.v.double()
        ks = self.ks.roll(1, -1) if shifted else self.ks
        return self.k.float().double() * ks.double().unsqueeze(-1), self.v.float().double() * self.vs.double().unsqueeze(-1)

    def on_gpu(self, o):
        if self.fmt == "none":
            return self.k.cuda(), self.v.cuda()
        four = (1,) * (4 - self.k.dim()) + tuple(self.k.shape)
        return o.QuantKV(self.k.view(four).cuda(), self.ks.view(four[:3]).cuda(), self.v.view(four).cuda(), self.vs.view(four[:3]).cuda())


class Case:
    def __init__(self, B, Hq, Hkv, n, P, S, d, dtype, fmt=("none", "none"), causal=False, lens=None, qscale=1.0, seed=0):
        self.B, self.Hq, self.Hkv, self.n, self.P, self.S, self.d = B, Hq, Hkv, n, P, S, d
        self.dtype, self.fmt, self.causal = dtype, fmt, causal
        self.lens = [S] * B if lens is None else list(lens)
        self.ragged = lens is not None
        self.q = randn((B, n, Hq, d), seed, qscale).to(dtype).transpose(1, 2)
        self.pre = Part((Hkv, P, d), fmt[0], dtype, seed + 100) if P else None
        self.own = Part((B, Hkv, S, d), fmt[1], dtype, seed + 200) if S else None

    def run(self, o):
        lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda") if self.ragged else None
        return o.shared_prefix_attention(self.q.cuda(), self.pre and self.pre.on_gpu(o), self.own and self.own.on_gpu(o),
                                         own_len=lens, causal=self.causal)

    def exact(self, device="cpu", shifted=False, drop=None, late=0):
        """-> out (B, n, Hq*d), and per element sum p |v|, largest sum |q_i k_i| * scale over the row's keys, largest |v|.
        drop: (part, first, end) keys left out; late: the causal limit is off by so many keys."""
        B, Hq, Hkv, n, d = self.B, self.Hq, self.Hkv, self.n, self.d
        scale = d ** -0.5
        none = torch.zeros((Hkv, 0, d), dtype=torch.float64)
        kp, vp = (t.to(device) for t in (self.pre.numbers(shifted) if self.pre else (none, none)))
        ko, vo = (t.to(device) for t in (self.own.numbers(shifted) if self.own else (none.expand(B, Hkv, 0, d),) * 2))
        out, av, vm = (torch.zeros((B, n, Hq, d), dtype=torch.float64, device=device) for _ in range(3))
        qk = torch.zeros((B, n, Hq, 1), dtype=torch.float64, device=device)
        for b in range(B):
            L = min(max(self.lens[b], 0), self.S)
            for h in range(Hq):
                hk = h // (Hq // Hkv)
                k, v = torch.cat([kp[hk], ko[b, hk, :L]]), torch.cat([vp[hk], vo[b, hk, :L]])
                if not len(k):
                    continue
                q = self.q[b, h].to(device).double()
                s = q @ k.T * scale
                at = torch.arange(len(k), device=device)
                if self.causal:
                    i = torch.arange(n, device=device)[:, None]
                    s = s.masked_fill(at[None] >= self.P + (L - n + 1 + i + late).clamp_min(0), -math.inf)
                if drop:
                    first, end = (x + (self.P if drop[0] == "own" else 0) for x in drop[1:])
                    s = s.masked_fill((at >= first) & (at < end), -math.inf)
                p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
                out[b, :, h], av[b, :, h], vm[b, :, h] = p @ v, p @ v.abs(), v.abs().max()
                qk[b, :, h] = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * scale
        flat = lambda t: t.expand(B, n, Hq, d).reshape(B, n, Hq * d)
        return flat(out), flat(av), flat(qk), flat(vm)

    def tolerance(self, out, av, qk, vm):
        """u: half a step of the call's type, o: the exact output, A = sum p |v|.
          probabilities are rounded once each: |sum p delta (v - o)| <= u (A + |o|), whichever sum they are divided by
          values that were codes are rounded once each: u A;  the output: u |o|;  products of these errors: (1 + 4 u)
          a logit is f32: d + 8 roundings of at most F32 sum|q k| (keys are exact in either form), and the exponential is good
          to 2^-20: e relative for every weight, e (A + |o|)
          sums over N keys, their parts and their rescalings: (N + 64) F32 of A, and of the row sum
          half precision: a probability below 2^-20 of the largest has an absolute error of 2^-31 of it: N 2^-31 max|v| (its
          values below 2^-14 likewise: 2^-25 each)"""
        u, N = HALF[self.dtype], self.P + self.S
        coded = u if self.fmt != ("none", "none") else 0.0
        e = torch.expm1(2 * (qk * (self.d + 8) * F32 + 2.0 ** -20)) + (N + 64) * F32
        tol = (1 + 4 * u) * (u * (av + out.abs()) + coded * av + u * out.abs()) + e * (av + out.abs())
        if self.dtype == torch.float16:
            tol = tol + N * 2.0 ** -31 * vm + 2.0 ** -24
        return tol + 1e-30


BF16, F16 = torch.bfloat16, torch.float16
CODES = [("int8", "int8"), ("e4m3", "e4m3"), ("int8", "none"), ("none", "e4m3")]

# what the tests run: decoding on grouped heads, drafted tokens in causal order, the network's layers behind one stored entry,
# heads of each class, few keys.  Causal cases have queries and keys of a size at which single keys count.
CASES = {}
for _t, _name in ((BF16, "bf16"), (F16, "f16")):
    for _f in CODES + [("none", "none")]:
        _tag = "%s %s/%s " % ((_name,) + _f)
        CASES[_tag + "decode"] = dict(B=4, Hq=8, Hkv=2, n=1, P=333, S=70, d=128, dtype=_t, fmt=_f, lens=[70, 67, 64, 1])
        CASES[_tag + "draft"] = dict(B=3, Hq=8, Hkv=4, n=5, P=133, S=70, d=80, dtype=_t, fmt=_f, causal=True, lens=[70, 33, 5], qscale=3.0)
        CASES[_tag + "image"] = dict(B=2, Hq=2, Hkv=2, n=200, P=333, S=0, d=40, dtype=_t, fmt=_f)
        CASES[_tag + "causal prompt"] = dict(B=2, Hq=4, Hkv=2, n=90, P=20, S=90, d=64, dtype=_t, fmt=_f, causal=True, qscale=3.0)
        CASES[_tag + "many sequences"] = dict(B=40, Hq=4, Hkv=2, n=1, P=150, S=9, d=64, dtype=_t, fmt=_f, lens=[b % 10 for b in range(40)])
        CASES[_tag + "wide heads"] = dict(B=2, Hq=2, Hkv=1, n=40, P=65, S=33, d=160, dtype=_t, fmt=_f, lens=[33, 0])
        CASES[_tag + "widest heads"] = dict(B=1, Hq=2, Hkv=2, n=3, P=129, S=31, d=256, dtype=_t, fmt=_f)
        CASES[_tag + "split keys"] = dict(B=1, Hq=2, Hkv=2, n=1, P=2500, S=700, d=64, dtype=_t, fmt=_f, qscale=2.0)
