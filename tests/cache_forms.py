"""Which kernel a call of the cache operators runs, by the rules of the library itself (hoard_kv_attention_form,
hoard_kv_choose_form): a test that is meant for one of them says so, whatever becomes of the rules' costs."""
import ctypes
import math

import torch

from hoard_b200 import cache
from tests import cache_ref as ref

MMA, TC, TC_WHOLE = "mma", "tc", "tc, no splits"
CHOOSE = ("one CTA", "cluster forms the keys", "cluster")

# head layout, tokens and past of a case for each kernel of the dense attention. 132 query rows over 38 KV heads: 76 tiles of
# 128 rows, the second of each head with four, and no room for splits
SHAPES = [
    dict(n_head=8, n_kv=2, hd=128, m=20, n_past=900, kernel=MMA),
    dict(n_head=8, n_kv=2, hd=128, m=20, n_past=4000, kernel=TC),
    dict(n_head=152, n_kv=38, hd=64, m=33, n_past=1000, kernel=TC_WHOLE)]


def attention_form(n_head, n_kv, hd, kt, rows, m, n_past, blocks=-1, block=0, acc=False):
    """(kernel, rows of a tile, splits, joined by a cluster)"""
    d = cache.Desc(n_head, n_kv, hd, cache.KV_TYPES[kt], rows, m, m if acc else 0, block, 0, 0, 1 / math.sqrt(hd))
    form = (ctypes.c_int32 * 4)()
    f = cache._kv().hoard_kv_attention_form
    f.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4 + [ctypes.c_void_p]
    assert f(ctypes.addressof(d), m, n_past, blocks, int(acc), ctypes.addressof(form)) == 0
    kernel = MMA if not form[0] else TC if form[2] > 1 else TC_WHOLE
    return kernel, form[1], form[2], bool(form[3])


def choose_form(n_cand, problems):
    f = cache._kv().hoard_kv_choose_form
    f.argtypes = [ctypes.c_int] * 2
    return CHOOSE[f(n_cand, problems)]


def kernel_of(s, kt):
    return attention_form(s["n_head"], s["n_kv"], s["hd"], kt, s["n_past"] + s["m"], s["m"], s["n_past"])[0]


def attention64(q, k, v, n_past, vis=None, gate=None, scale=None):
    """cache_ref.attention on the inputs' device: out [m][n_head][hd] in 64 bits. Every token has to see finite rows only."""
    m, n_head, hd = q.shape
    n_kv = k.shape[1]
    g, n = n_head // n_kv, n_past + m
    own = ref.visibility(vis, m).to(q.device)
    x = torch.einsum("tkgd,jkd->ktgj", q.double().view(m, n_kv, g, hd), k[:n].double()) * (1 / math.sqrt(hd) if scale is None else scale)
    x[..., n_past:].masked_fill_(~own[None, :, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    out = torch.einsum("ktgj,jkd->tkgd", p, v[:n].double()).reshape(m, n_head, hd)
    return out if gate is None else out * torch.sigmoid(gate.double())
