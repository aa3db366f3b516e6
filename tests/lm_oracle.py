"""The language-model operators in 64 bits, and how far a kernel that computes in fp32 may be off them.

A rounding to a type is off by at most half a step, ``finfo.eps / 2`` relative to the value, or half the smallest
subnormal.  U = 2^-24 is that half step in fp32.
"""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of subnormal values."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what):
    """|got - want| <= bound, value by value; NaN and infinities have to agree."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), '%s: NaN at other places' % what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), '%s: other infinities' % what
    fine = ~(want.isnan() | inf)
    bound = torch.as_tensor(bound, dtype=torch.float64).detach().cpu().expand_as(want)
    off = (got - want).abs()[fine] - bound[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, '%s: %.3g over its bound %.3g' % (
        what, float(off.max()), float(bound[fine][off.argmax()]))


# ------------------------------------------------------------------------------------------------------- embedding
def embedding_grad(dy, tokens, vocab, scale, padding=None):
    """Sum for each token, and the bound of an fp32 sum of m terms in any order, its product with the factor (itself
    rounded to fp32) and one rounding to the type: ((m - 1) + 2) U sum|x| |scale| + half a step of the result."""
    ids, rows = tokens.reshape(-1).long(), dy.detach().reshape(-1, dy.shape[-1]).double()
    if padding is not None:
        keep = ids != padding
        ids, rows = ids[keep], rows[keep]
    want = torch.zeros(vocab, rows.shape[1], dtype=torch.float64, device=dy.device).index_add_(0, ids, rows)
    mass = torch.zeros_like(want).index_add_(0, ids, rows.abs())
    m = torch.bincount(ids, minlength=vocab).double().unsqueeze(1)
    want *= scale
    bound = (m + 2) * U * mass * abs(scale) * (1 + 1e-6) + half_step(dy.dtype) * want.abs() * (1 + 1e-3) + tiny(dy.dtype)
    return want, bound


# ---------------------------------------------------------------------------------------------------- log probabilities
class Rows:
    """One set of rows in 64 bits with the error bounds of an fp32 evaluation.

    An exponential of d = z - m is off by (|d| + 4) U relatively (the difference rounds by |d| U, the function by two
    units, two steps of 2^-23), a sum of V positive terms in 128 or more strands by (V / 128 + 20) U (strand, tree and the
    rescaling of the parts).  Weighted with the terms, s is off by es = (V / 128 + 24 + u1) U with u1 = sum e |d| / s, and
    u = sum e d by (V / 128 + 26) U |u| + U sum e d^2.
    """

    def __init__(self, logits, tokens, ignore=-100):
        self.z = z = logits.detach().reshape(-1, logits.shape[-1]).double()
        self.ids = tokens.reshape(-1).long()
        self.ignore, self.vocab = ignore, z.shape[1]
        self.pad = self.ids == ignore
        self.bad = ~self.pad & ((self.ids < 0) | (self.ids >= self.vocab))
        m = z.amax(1, keepdim=True)
        self.fine = m.isfinite().squeeze(1)
        d = torch.where(m.isfinite(), z - m, torch.zeros_like(z))
        e = d.exp()
        d = torch.where(e > 0, d, torch.zeros_like(d))
        s = e.sum(1)
        self.m, self.ln_s = m.squeeze(1), s.log()
        self.u = (e * d).sum(1)
        k = self.vocab / 128 + 26
        self.es = (k + self.u.abs() / s) * U
        self.eu = (k * self.u.abs() + (e * d * d).sum(1)) / s * U
        self.d, self.e, self.s = d, e, s

    def _rows(self, v, padded=0.0):
        v = torch.where(self.fine & ~self.bad, v, torch.full_like(v, math.nan))
        return torch.where(self.pad, torch.full_like(v, padded), v)

    def logprob_of(self, ids):
        dt = self.z.gather(1, ids) - self.m.unsqueeze(1)
        lp = dt - self.ln_s.unsqueeze(1)
        bound = self.es.unsqueeze(1) + U * (dt.abs() + 4 * self.ln_s.unsqueeze(1) + lp.abs())
        return lp, torch.where(bound.isfinite(), bound, torch.zeros_like(bound))

    def logprob(self):
        lp, bound = self.logprob_of(self.ids.clamp(0, self.vocab - 1).unsqueeze(1))
        return self._rows(lp.squeeze(1)), bound.squeeze(1)

    def entropy(self):
        h = self.ln_s - self.u / self.s
        # ln s (error es and two units), the quotient (errors of u and s, one rounding), the difference
        bound = self.es * (1 + (self.u / self.s).abs()) + self.eu + U * (4 * self.ln_s + 2 * (self.u / self.s).abs() + h.abs())
        h = torch.where(self.fine, h, torch.full_like(h, math.nan))                    # needs no token
        return torch.where(self.pad, torch.zeros_like(h), h), bound

    def top(self, k):
        key = self.z.clone()
        key[key.isnan()] = math.inf                                                    # NaN above everything
        nan_first = torch.where(self.z.isnan(), 1, 0)
        order = torch.argsort(key, dim=1, descending=True, stable=True)
        order = order.gather(1, torch.argsort(nan_first.gather(1, order), dim=1, descending=True, stable=True))[:, :k]
        lp, bound = self.logprob_of(order)
        lp = torch.where(self.fine.unsqueeze(1), lp, torch.full_like(lp, math.nan))
        lp = torch.where(self.pad.unsqueeze(1), torch.zeros_like(lp), lp)
        return lp, bound, order.masked_fill(self.pad.unsqueeze(1), -1)

    def grad(self, g1, g2, dtype):
        """Gradient of sum g1 logprob + g2 entropy: p is off by the error of ln s, of two differences and of the
        exponential; the bracket by the errors of ln p and H; the products round a few times, the result once more."""
        g1, g2 = g1.double().unsqueeze(1), g2.double().unsqueeze(1)
        lp = self.d - self.ln_s.unsqueeze(1)
        p = self.e / self.s.unsqueeze(1)
        h, eh = self.entropy()
        h, eh = h.unsqueeze(1), eh.unsqueeze(1)
        elp = self.es.unsqueeze(1) + U * (self.d.abs() + 4 * self.ln_s.unsqueeze(1) + 2 * lp.abs())
        inner = g1 + g2 * (lp + h)
        want = -p * inner
        at = torch.arange(len(self.z), device=self.z.device)
        valid = ~self.pad & ~self.bad
        want[at[valid], self.ids[valid]] += g1.squeeze(1)[valid]
        bound = p * ((elp + 4 * U) * (g1.abs() + g2.abs() * (lp.abs() + h.abs())) + g2.abs() * (elp + eh)) + \
            4 * U * (p * (g1.abs() + g2.abs() * (lp.abs() + h.abs())) + g1.abs())
        want = torch.where((self.fine & ~self.bad).unsqueeze(1), want, torch.full_like(want, math.nan))
        want = torch.where(self.pad.unsqueeze(1), torch.zeros_like(want), want)
        bound = bound * (1 + half_step(dtype)) + half_step(dtype) * want.nan_to_num().abs() + tiny(dtype) + 2 * tiny(torch.float32)
        return want, bound
