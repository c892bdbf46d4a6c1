"""A minimal decode driver around the MoE path: hoard's per-token schedule (src/run_moe_stream.cpp:
295-472) with every step on the device.

    graph E   x = token_embd[token]                                            (hoard_hx_embed)
    per layer (graph A, attention part; then the MoE layer):
              cur = RMSNorm(x) * attn_norm
              q, k, v = Wq cur, Wk cur, Wv cur          (Q4_K / Q6_K . Q8_K(cur), hoard_hx_gemv)
              QK RMSNorm: over the whole projection (OLMoE) or per head (Qwen3)
              NEOX RoPE of q, k at position p; k, v into the f16/bf16 KV cache (hoard_hx_rope_store)
              att = softmax(q k^T / sqrt(head_dim)) v over positions 0..p     (hoard_hx_attention)
              ffn_inp = Wo att + x
              x = ffn_inp + sum_j w_j FFN_j(RMSNorm(ffn_inp) * ffn_norm)       (hoard_moe_layers)
    head      logits = W_out (RMSNorm(x) * output_norm); next = argmax         (hoard_hx_argmax)

Prompt tokens run through the same step one at a time, as in hoard; generation starts from the
logits of the last prompt token. Models come from a GGUF file (`DecodeModel.from_gguf`) or from
seeded tensors generated on the device (`seeded_tensors`, the benchmark configurations' weights:
N(0, 0.02), Q4_K_M types). The MoE layers use all experts HBM-resident (T = 1: the persistent
decode kernel).

Beside the plain step there are three forms of the attention over the cache (hoard_b200/cache.py):
`tree_generate` verifies a tree of drafted tokens in one forward (`forward_tree`); `blocks=BlockChoice(..)` lets every
token attend the first, the last and the best-scoring blocks of a long cache; `budget=CacheBudget(..)` keeps a bounded
number of cache rows per KV head, evicting the positions with the least accumulated attention weight. Positions beyond
what the one-CTA-per-head attention holds in shared memory (and captured steps of contexts beyond it) run through the split
attention of the same module."""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import numpy as np
import torch

from hoard_b200 import cache, moe, quant
from hoard_b200.moe import HoardError, _ptr, _stream, lib

Q4_K, Q6_K, F32 = quant.Q4_K, quant.Q6_K, 0
KV_TYPES = {torch.float16: 1, torch.bfloat16: 30}     # KV cache element -> HOARD_TYPE_F16 / HOARD_TYPE_BF16
MAX_BATCH = 16          # tokens of one batched (verify) forward
QK_MODE = {"": 0, "full": 1, "head": 2}


@dataclass
class BlockChoice:
    """Attention over blocks of `block` cache rows: the first n_sink, the last n_local and the n_sel best-scoring others
    for each token and KV head."""
    block: int = 64
    n_sink: int = 1
    n_local: int = 4
    n_sel: int = 32

    def leaves_out(self, rows: int) -> bool:
        """Whether a past of up to `rows` rows can have blocks that a token does not attend."""
        return self.n_sink + self.n_local + self.n_sel < -(-rows // self.block)


@dataclass
class CacheBudget:
    """A bounded cache: when n_keep + n_slack rows are filled, each KV head keeps n_keep of them -- the first n_sink and
    the last n_recent positions, then those with the largest accumulated attention weight."""
    n_keep: int
    n_slack: int = 256
    n_sink: int = 4
    n_recent: int = 128

    @property
    def rows(self) -> int:
        return self.n_keep + self.n_slack


def plain_attention_rows(head_dim: int) -> int:
    """Most positions that hoard_hx_attention takes: their scores share 200 KiB of shared memory with q and the partial sums of
    its 512 threads (256 where rows are no multiple of 16 bytes). 0: it does not take the head_dim."""
    if head_dim < 1 or 256 % head_dim:
        return 0
    groups = 512 // (head_dim // 8) if head_dim % 8 == 0 else 256 // head_dim
    return 200 * 1024 // 4 - head_dim - groups * head_dim


def _iarr(vals):
    return (ctypes.c_int * len(vals))(*vals)


def _parr(ptrs):
    return (ctypes.c_void_p * len(ptrs))(*ptrs)

_bound = False


def _hx():
    global _bound
    L = lib()
    if not _bound:
        vp, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        L.hoard_hx_repack.argtypes = [i32, vp, vp, i64, vp]
        L.hoard_hx_embed.argtypes = [i32, vp, i32, i64, vp, vp, vp]
        L.hoard_hx_rmsnorm.argtypes = [vp, i32, i32, f32, vp, vp, vp]
        L.hoard_hx_q8_bytes.argtypes = [i32]
        L.hoard_hx_q8_bytes.restype = i64
        L.hoard_hx_quant_q8.argtypes = [vp, i32, vp, vp]
        L.hoard_hx_gemv.argtypes = [i32, vp, i32, i32, vp, vp, vp, vp]
        L.hoard_hx_rope_store.argtypes = [vp, vp, vp, i32, i32, i32, i32, f32, vp, vp, i32, vp]
        L.hoard_hx_attention.argtypes = [vp, vp, vp, i32, i32, i32, i32, f32, vp, i32, vp]
        L.hoard_hx_argmax.argtypes = [vp, i32, vp, vp]
        L.hoard_hx_embed_at.argtypes = [i32, vp, i32, i64, vp, vp, vp, vp]
        L.hoard_hx_rope_store_at.argtypes = [vp, vp, vp, i32, i32, i32, vp, i32, f32, vp, vp, i32, vp]
        L.hoard_hx_attention_at.argtypes = [vp, vp, vp, i32, i32, i32, vp, i32, f32, vp, i32, vp]
        L.hoard_hx_argmax_at.argtypes = [vp, i32, vp, vp, i32, vp]
        L.hoard_hx_rmsnorm_q8.argtypes = [vp, i32, f32, vp, vp, vp]
        L.hoard_hx_gemv_multi.argtypes = [i32, vp, vp, vp, i32, vp, vp, vp, vp]
        L.hoard_hx_qknorm_rope_store.argtypes = [vp, vp, vp, vp, vp, i32, f32, i32, i32, i32, i32, f32, vp, vp, vp, i32,
                                                 vp]
        L.hoard_hx_qknorm_rope_store_at.argtypes = [vp, vp, vp, vp, vp, i32, f32, i32, i32, i32, vp, i32, f32, vp, vp,
                                                   vp, i32, vp]
        L.hoard_hx_qknorm_rope_store_ex.argtypes = [vp, vp, vp, vp, vp, i32, f32, i32, i32, i32, i32, i32, i32, vp, i32,
                                                   f32, vp, vp, vp, i32, vp]
        L.hoard_hx_attention_ex.argtypes = [vp, vp, vp, i32, i32, i32, i32, vp, f32, vp, i32, vp, i32, vp]
        L.hoard_hx_gdn_step.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, f32, i32, vp, vp, vp]
        _bound = True
    return L


def _ok(rc: int, what: str):
    if rc != 0:
        raise HoardError(rc, f"{what} failed ({lib().hoard_strerror(rc).decode()})")


@dataclass
class ModelConfig:
    """Hyper-parameters and GGUF tensor types of a seeded model (Q4_K_M: attn q/k/o and the
    embedding Q4_K, attn v and the lm-head Q6_K, expert gate/up Q4_K, expert down Q6_K on even and
    Q4_K on odd layers)."""
    arch: str
    n_layer: int
    n_embd: int
    n_head: int
    n_head_kv: int
    head_dim: int
    n_expert: int
    n_expert_used: int
    n_ff: int
    n_vocab: int
    freq_base: float
    eps: float
    qk_norm: str            # "full" (OLMoE: over the whole projection), "head" (Qwen3) or ""
    norm_topk: bool
    # hybrid models (Qwen3-Next, src/run_qwen35.cpp:472-553): every full_attn_interval-th layer is gated
    # full attention (fused q + sigmoid output gate, NEOX RoPE on the first rope_dim values of a head),
    # the others gated delta-net; a gated shared expert of n_ff_shexp
    n_ff_shexp: int = 0
    full_attn_interval: int = 0     # 0: every layer is full attention
    attn_gate: bool = False
    rope_dim: int = 0               # 0: head_dim
    ssm_d_state: int = 0            # delta-net head dim (key = value)
    ssm_n_group: int = 0            # key heads
    ssm_dt_rank: int = 0            # value heads
    ssm_d_conv: int = 0             # causal conv taps

    def down_type(self, il: int) -> int:
        return Q6_K if il % 2 == 0 else Q4_K

    def is_recurrent(self, il: int) -> bool:
        return self.full_attn_interval > 0 and (il + 1) % self.full_attn_interval != 0

    def ffn_norm_name(self) -> str:
        return "post_attention_norm.weight" if self.full_attn_interval > 0 else "ffn_norm.weight"

    @property
    def n_rot(self) -> int:
        return self.rope_dim or self.head_dim

    @property
    def conv_dim(self) -> int:
        return (2 * self.ssm_n_group + self.ssm_dt_rank) * self.ssm_d_state


C1_OLMOE = ModelConfig("olmoe", 16, 2048, 16, 16, 128, 64, 8, 1024, 50304, 1e4, 1e-5, "full", False)
C3_QWEN3 = ModelConfig("qwen3moe", 48, 2048, 32, 4, 128, 128, 8, 768, 151936, 1e6, 1e-6, "head", True)
C5_QWEN3NEXT = ModelConfig("qwen3next", 48, 2048, 16, 2, 256, 512, 10, 512, 151936, 1e7, 1e-6, "head", True,
                           n_ff_shexp=512, full_attn_interval=4, attn_gate=True, rope_dim=64, ssm_d_state=128,
                           ssm_n_group=16, ssm_dt_rank=32, ssm_d_conv=4)


def seeded_tensors(cfg: ModelConfig, seed: int, device) -> dict:
    """Every tensor of a seeded model, named as in hoard's GGUFs, on `device`:
    name -> (ggml type, ne (GGUF order), tensor: uint8 raw blocks or f32)."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    H, hd, E, I = cfg.n_embd, cfg.head_dim, cfg.n_expert, cfg.n_ff
    nq, nkv = cfg.n_head * hd, cfg.n_head_kv * hd

    def w(n_out, k_in, qt):
        return quant.quantize(torch.randn(n_out, k_in, generator=g, device=device) * 0.02, qt)

    def norm(n):
        return (1.0 + 0.1 * torch.randn(n, generator=g, device=device)).float()

    t = {"token_embd.weight": (Q4_K, (H, cfg.n_vocab), w(cfg.n_vocab, H, Q4_K)),
         "output_norm.weight": (F32, (H,), norm(H)),
         "output.weight": (Q6_K, (H, cfg.n_vocab), w(cfg.n_vocab, H, Q6_K))}
    for il in range(cfg.n_layer):
        b = f"blk.{il}."
        t[b + "attn_norm.weight"] = (F32, (H,), norm(H))
        if cfg.is_recurrent(il):
            D, Hk, Hv = cfg.ssm_d_state, cfg.ssm_n_group, cfg.ssm_dt_rank
            cd, vd = cfg.conv_dim, Hv * D
            t[b + "attn_qkv.weight"] = (Q4_K, (H, cd), w(cd, H, Q4_K))
            t[b + "attn_gate.weight"] = (Q4_K, (H, vd), w(vd, H, Q4_K))
            t[b + "ssm_ba.weight"] = (Q4_K, (H, 2 * Hv), w(2 * Hv, H, Q4_K))
            t[b + "ssm_conv1d.weight"] = (F32, (cfg.ssm_d_conv, cd),
                                          (torch.randn(cd, cfg.ssm_d_conv, generator=g, device=device) * 0.3).float())
            t[b + "ssm_dt.bias"] = (F32, (Hv,), (torch.randn(Hv, generator=g, device=device) * 0.5).float())
            # ssm_a = -exp(A_log), A_log ~ U(0, log 16)
            t[b + "ssm_a"] = (F32, (Hv,), (-torch.exp(torch.rand(Hv, generator=g, device=device) * math.log(16.0))).float())
            t[b + "ssm_norm.weight"] = (F32, (D,), norm(D))
            t[b + "ssm_out.weight"] = (Q4_K, (vd, H), w(H, vd, Q4_K))
        else:
            nqp = 2 * nq if cfg.attn_gate else nq
            t[b + "attn_q.weight"] = (Q4_K, (H, nqp), w(nqp, H, Q4_K))
            t[b + "attn_k.weight"] = (Q4_K, (H, nkv), w(nkv, H, Q4_K))
            t[b + "attn_v.weight"] = (Q6_K, (H, nkv), w(nkv, H, Q6_K))
            t[b + "attn_output.weight"] = (Q4_K, (nq, H), w(H, nq, Q4_K))
            if cfg.qk_norm == "full":
                t[b + "attn_q_norm.weight"] = (F32, (nq,), norm(nq))
                t[b + "attn_k_norm.weight"] = (F32, (nkv,), norm(nkv))
            elif cfg.qk_norm == "head":
                t[b + "attn_q_norm.weight"] = (F32, (hd,), norm(hd))
                t[b + "attn_k_norm.weight"] = (F32, (hd,), norm(hd))
        t[b + cfg.ffn_norm_name()] = (F32, (H,), norm(H))
        t[b + "ffn_gate_inp.weight"] = (F32, (H, E), (torch.randn(E, H, generator=g, device=device) * 0.02).float())
        dt = cfg.down_type(il)
        t[b + "ffn_gate_exps.weight"] = (Q4_K, (H, I, E), quant.synth_experts(E, I, H, Q4_K, seed * 1000 + 3 * il, device))
        t[b + "ffn_up_exps.weight"] = (Q4_K, (H, I, E), quant.synth_experts(E, I, H, Q4_K, seed * 1000 + 3 * il + 1, device))
        t[b + "ffn_down_exps.weight"] = (dt, (I, H, E), quant.synth_experts(E, H, I, dt, seed * 1000 + 3 * il + 2, device))
        if cfg.n_ff_shexp:
            Is = cfg.n_ff_shexp
            t[b + "ffn_gate_shexp.weight"] = (Q4_K, (H, Is), w(Is, H, Q4_K))
            t[b + "ffn_up_shexp.weight"] = (Q4_K, (H, Is), w(Is, H, Q4_K))
            t[b + "ffn_down_shexp.weight"] = (Q6_K, (Is, H), w(H, Is, Q6_K))
            t[b + "ffn_gate_inp_shexp.weight"] = (F32, (H,), (torch.randn(H, generator=g, device=device) * 0.02).float())
    return t


def write_gguf(path: str, cfg: ModelConfig, tensors: dict):
    from hoard_b200 import gguf_io as gi
    w = gi.GGUFWriter(cfg.arch)
    a = cfg.arch
    w.add(f"{a}.block_count", cfg.n_layer)
    w.add(f"{a}.embedding_length", cfg.n_embd)
    w.add(f"{a}.attention.head_count", cfg.n_head)
    w.add(f"{a}.attention.head_count_kv", cfg.n_head_kv)
    w.add(f"{a}.attention.key_length", cfg.head_dim)
    w.add(f"{a}.expert_feed_forward_length", cfg.n_ff)
    w.add(f"{a}.expert_count", cfg.n_expert)
    w.add(f"{a}.expert_used_count", cfg.n_expert_used)
    w.add(f"{a}.rope.freq_base", float(cfg.freq_base))
    w.add(f"{a}.attention.layer_norm_rms_epsilon", float(cfg.eps))
    for name, (ty, ne, data) in tensors.items():
        w.add_tensor(name, ne, ty, data.detach().cpu().numpy())
    w.write(path)


def config_from_hparams(hp) -> ModelConfig:
    return ModelConfig(hp.arch, hp.n_layer, hp.n_embd, hp.n_head, hp.n_head_kv, hp.head_dim, hp.n_expert,
                       hp.n_expert_used, hp.n_ff, hp.n_vocab, hp.freq_base, hp.eps,
                       "" if not hp.has_qk_norm else ("head" if hp.qk_perhead else "full"), hp.norm_topk)


class DecodeModel:
    def __init__(self, cfg: ModelConfig, tensors: dict, device: int = 0, max_ctx: int = 512, eos_id: int = -1,
                 kv_dtype=torch.float16, max_batch: int = MAX_BATCH, blocks: BlockChoice | None = None,
                 budget: CacheBudget | None = None):
        """tensors: name -> (ggml type, ne, array or tensor of raw bytes / f32 values), host or device.
        kv_dtype: torch.float16 or torch.bfloat16 elements of the KV cache. max_batch: most tokens of a batched
        forward (verify pass), up to 64. blocks / budget: the block-sparse or the bounded form of the cache."""
        if kv_dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("kv_dtype must be torch.float16 or torch.bfloat16")
        if not 1 <= max_batch <= cache.MAX_TOKENS:
            raise ValueError(f"max_batch must be 1..{cache.MAX_TOKENS}")
        if blocks is not None and budget is not None:
            raise ValueError("blocks of the cache need its rows in the order of positions: not with a budget")
        if blocks is not None and max_ctx < blocks.block:
            raise ValueError("max_ctx holds one block at least")
        if budget is not None and not (0 <= budget.n_sink and 0 <= budget.n_recent and budget.n_slack >= 1
                                       and budget.n_sink + budget.n_recent < budget.n_keep):
            raise ValueError("a budget keeps more rows than its first and last positions, and has slack")
        self.max_batch, self.blocks, self.budget = max_batch, blocks, budget
        self.cfg, self.device, self.max_ctx, self.eos_id = cfg, device, max_ctx, eos_id
        self.kv_type = KV_TYPES[kv_dtype]
        dev = self.dev = torch.device("cuda", device)
        _hx()
        H, hd = cfg.n_embd, cfg.head_dim
        self.nq, self.nkv = cfg.n_head * hd, cfg.n_head_kv * hd

        def raw(name):
            ty, ne, data = tensors[name]
            t = torch.as_tensor(np.asarray(data)) if not isinstance(data, torch.Tensor) else data
            return ty, t.contiguous().to(dev)

        def plane(name):
            ty, t = raw(name)
            out = torch.empty_like(t, dtype=torch.uint8)
            nblk = t.numel() // quant.row_bytes(ty, 256)
            _ok(_hx().hoard_hx_repack(ty, _ptr(t), _ptr(out), nblk, _stream(None)), "repack")
            return ty, out

        def f32(name):
            ty, t = raw(name)
            assert ty == F32
            return t.view(torch.float32) if t.dtype == torch.uint8 else t.float()

        self.embd_type, self.embd = raw("token_embd.weight")
        self.out_norm = f32("output_norm.weight")
        self.out_type, self.out_w = plane("output.weight")
        self.nqp = 2 * self.nq if cfg.attn_gate else self.nq      # q projection rows (+ the output gate)
        hybrid = cfg.full_attn_interval > 0
        self.gdn_vd = cfg.ssm_dt_rank * cfg.ssm_d_state
        self.layers = []
        for il in range(cfg.n_layer):
            b = f"blk.{il}."
            L = {"attn_norm": f32(b + "attn_norm.weight"), "recurrent": cfg.is_recurrent(il)}
            if L["recurrent"]:
                L.update({"qkv": plane(b + "attn_qkv.weight"), "z": plane(b + "attn_gate.weight"),
                          "ba": plane(b + "ssm_ba.weight"), "conv_w": f32(b + "ssm_conv1d.weight"),
                          "dt_bias": f32(b + "ssm_dt.bias"), "ssm_a": f32(b + "ssm_a"),
                          "ssm_norm": f32(b + "ssm_norm.weight"), "o": plane(b + "ssm_out.weight")})
                L["qkv_types"] = _iarr([L[m][0] for m in ("qkv", "z", "ba")])
                L["qkv_w"] = _parr([L[m][1].data_ptr() for m in ("qkv", "z", "ba")])
            else:
                L.update({"q": plane(b + "attn_q.weight"), "k": plane(b + "attn_k.weight"),
                          "v": plane(b + "attn_v.weight"), "o": plane(b + "attn_output.weight")})
                if cfg.qk_norm:
                    L["q_norm"], L["k_norm"] = f32(b + "attn_q_norm.weight"), f32(b + "attn_k_norm.weight")
                L["qkv_types"] = _iarr([L[m][0] for m in ("q", "k", "v")])
                L["qkv_w"] = _parr([L[m][1].data_ptr() for m in ("q", "k", "v")])
            self.layers.append(L)
        # the MoE layers: all experts resident, T = 1
        types = [tuple(tensors[f"blk.{il}.ffn_{m}_exps.weight"][0] for m in ("gate", "up", "down"))
                 for il in range(cfg.n_layer)]
        sh_types = (Q4_K, Q4_K, Q6_K)
        if cfg.n_ff_shexp:
            sh_types = tuple(tensors[f"blk.0.ffn_{m}_shexp.weight"][0] for m in ("gate", "up", "down"))
        self.moe = moe.MoEContext(n_embd=H, n_expert=cfg.n_expert, n_expert_used=cfg.n_expert_used, n_ff=cfg.n_ff,
                                  n_layer=cfg.n_layer, norm_topk=cfg.norm_topk, eps=cfg.eps,
                                  gate_types=[t[0] for t in types], up_types=[t[1] for t in types],
                                  down_types=[t[2] for t in types], n_ff_shexp=cfg.n_ff_shexp, shexp_types=sh_types,
                                  max_tokens=max_batch, device=device)
        for il in range(cfg.n_layer):
            b = f"blk.{il}."
            self.moe.set_router(il, f32(b + "ffn_gate_inp.weight").view(cfg.n_expert, H), f32(b + cfg.ffn_norm_name()))
            mats = [raw(b + f"ffn_{m}_exps.weight")[1].view(cfg.n_expert, -1) for m in ("gate", "up", "down")]
            for e in range(cfg.n_expert):
                self.moe.upload_expert(il, e, mats[0][e], mats[1][e], mats[2][e])
            if cfg.n_ff_shexp:
                self.moe.set_shared(il, *(raw(b + f"ffn_{m}_shexp.weight")[1] for m in ("gate", "up", "down")),
                                    f32(b + "ffn_gate_inp_shexp.weight"))
        # activations, Q8_K workspaces, KV caches, delta-net states, token sequence
        z = lambda n: torch.zeros(n, dtype=torch.float32, device=dev)
        self.x, self.x2, self.cur = z(H), z(H), z(H)
        self.q, self.k, self.v, self.att = z(self.nqp), z(self.nkv), z(self.nkv), z(self.nq)
        self.logits = z(cfg.n_vocab)
        self.q_rot = z(self.nq)
        self.qkv_N = _iarr([self.nqp, self.nkv, self.nkv])
        self.qkv_y = _parr([self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr()])
        kq = max(H, self.nq, self.gdn_vd)
        self.q8 = torch.zeros(int(_hx().hoard_hx_q8_bytes(kq)), dtype=torch.uint8, device=dev)
        n_full = sum(1 for L in self.layers if not L["recurrent"])
        self.kv_index = {}
        for il, L in enumerate(self.layers):
            if not L["recurrent"]:
                self.kv_index[il] = len(self.kv_index)
        self.n_cache = budget.rows if budget else max_ctx         # rows of a layer's cache
        self.kc = torch.zeros(max(1, n_full), self.n_cache, self.nkv, dtype=kv_dtype, device=dev)
        self.vc = torch.zeros_like(self.kc)
        # the split attention: blocks, budgets, positions beyond the one-CTA attention's, and (made when first used) trees
        self._ops_args = dict(n_head=cfg.n_head, n_head_kv=cfg.n_head_kv, head_dim=hd, kv_dtype=kv_dtype,
                              max_rows=self.n_cache, block=blocks.block if blocks else 0, device=device)
        self.plain_rows = plain_attention_rows(hd)
        self.ops = None
        if blocks or budget or max_ctx > self.plain_rows:
            try:
                self.ops = cache.CacheOps(**self._ops_args)
            except HoardError:               # a head layout that only the one-CTA attention takes, up to its positions
                if blocks or budget:
                    raise
        self._tree_ops = None
        if blocks:
            self.bounds = torch.zeros(max(1, n_full), cfg.n_head_kv, self.n_cache // blocks.block, 2, hd, dtype=kv_dtype,
                                      device=dev)
        if budget:
            self.kv_acc = torch.zeros(max(1, n_full), cfg.n_head_kv, self.n_cache, dtype=torch.float32, device=dev)
            self.kv_pos = torch.zeros(max(1, n_full), cfg.n_head_kv, self.n_cache, dtype=torch.int32, device=dev)
            self.rows_dev = torch.zeros(1, dtype=torch.int32, device=dev)
        self.n_rows = 0         # filled rows of a bounded cache
        if hybrid:
            n_rec = cfg.n_layer - n_full
            self.gdn_qkv, self.gdn_z, self.gdn_ba = z(cfg.conv_dim), z(self.gdn_vd), z(2 * cfg.ssm_dt_rank)
            self.gdn_out = z(self.gdn_vd)
            self.gdn_N = _iarr([cfg.conv_dim, self.gdn_vd, 2 * cfg.ssm_dt_rank])
            self.gdn_y = _parr([self.gdn_qkv.data_ptr(), self.gdn_z.data_ptr(), self.gdn_ba.data_ptr()])
            self.gdn_ring = torch.zeros(n_rec, cfg.ssm_d_conv, cfg.conv_dim, dtype=torch.float32, device=dev)
            self.gdn_state = torch.zeros(n_rec, cfg.ssm_dt_rank, cfg.ssm_d_state, cfg.ssm_d_state, dtype=torch.float32,
                                         device=dev)
            self.rec_index = {il: i for i, il in enumerate(j for j, L in enumerate(self.layers) if L["recurrent"])}
        self.seq = torch.zeros(max_ctx + 1, dtype=torch.int32, device=dev)
        self.scratch_tok = torch.zeros(1, dtype=torch.int32, device=dev)
        self.all_pos = torch.arange(max_ctx, dtype=torch.int32, device=dev)
        self.pos_dev = torch.zeros(1, dtype=torch.int32, device=dev)
        self._graph = None
        torch.cuda.synchronize(dev)

    @classmethod
    def from_gguf(cls, path: str, device: int = 0, max_ctx: int = 512, kv_dtype=torch.float16, **kw):
        from hoard_b200 import gguf_io as gi
        g = gi.GGUFFile(path)
        hp = gi.read_hparams(g)
        tensors = {}
        for name, t in g.tensors.items():
            data = g.array(name) if t.type == F32 else g.data(name)
            tensors[name] = (t.type, t.ne, np.array(data))
        g.close()
        return cls(config_from_hparams(hp), tensors, device=device, max_ctx=max_ctx, eos_id=hp.eos_id,
                   kv_dtype=kv_dtype, **kw)

    def close(self):
        self.moe.close()

    # ---- one token: logits of position pos for token seq[pos]; argmax into `next_tok` ----
    def step(self, pos: int, next_tok: torch.Tensor, stream=None):
        c, hx, s = self.cfg, _hx(), _stream(stream)
        H = c.n_embd
        x, x2 = self.x, self.x2
        if self.budget:
            self._make_room(pos, stream)
        _ok(hx.hoard_hx_embed(self.embd_type, _ptr(self.embd), H, c.n_vocab, _ptr(self.seq[pos:pos + 1]), _ptr(x), s),
            "embed")
        for il, L in enumerate(self.layers):
            self._layer_attention(il, L, x, x2, hx, s, pos)
            self.moe.layers(il, 1, x2.view(1, H), stream=stream)
            x, x2 = x2, x
        _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x), H, c.eps, _ptr(self.out_norm), _ptr(self.q8), s), "rmsnorm_q8")
        _ok(hx.hoard_hx_gemv(self.out_type, _ptr(self.out_w), c.n_vocab, H, _ptr(self.q8), None, _ptr(self.logits), s),
            "gemv")
        _ok(hx.hoard_hx_argmax(_ptr(self.logits), c.n_vocab, _ptr(next_tok), s), "argmax")
        self.n_rows += 1

    # ---- bounded cache ----
    def _make_room(self, pos: int, stream=None):
        """Before the token at position pos is stored: a full cache is brought down to its budget."""
        b = self.budget
        if self.n_rows < b.rows:
            return
        for i in range(len(self.kv_index)):
            self.ops.evict(self._heads(self.kc[i]), self._heads(self.vc[i]), self.kv_acc[i], self.kv_pos[i], self.n_rows,
                           b.n_keep, n_sink=b.n_sink, recent_from=pos - b.n_recent, stream=stream)
        self.n_rows = b.n_keep

    def _heads(self, t):
        """A cache as [row][KV head][head_dim]."""
        return t.view(self.n_cache, self.cfg.n_head_kv, self.cfg.head_dim)

    def _layer_attention(self, il, L, x, x2, hx, s, pos=None, bufs=None):
        """Graph A's attention part of layer il: x2 = Wo att + x (or the delta-net block's output
        projection + x). pos None: the device position. bufs: (q, k, v, q_rot, att, qkv_y) of one token of
        a batch (default: the step's own)."""
        c = self.cfg
        H, hd = c.n_embd, c.head_dim
        if L["recurrent"]:
            self._layer_gdn(il, L, x, x2, hx, s, pos)
            return
        q, k, v, q_rot, att, qkv_y = bufs or (self.q, self.k, self.v, self.q_rot, self.att, self.qkv_y)
        kc, vc = self.kc[self.kv_index[il]], self.vc[self.kv_index[il]]
        _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x), H, c.eps, _ptr(L["attn_norm"]), _ptr(self.q8), s), "rmsnorm_q8")
        _ok(hx.hoard_hx_gemv_multi(3, L["qkv_types"], L["qkv_w"], self.qkv_N, H, _ptr(self.q8), None, qkv_y, s),
            "gemv qkv")
        mode = QK_MODE[c.qk_norm]
        qn, kn = (L["q_norm"], L["k_norm"]) if mode else (None, None)
        scale = 1.0 / math.sqrt(hd)
        qs = 2 * hd if c.attn_gate else hd           # a q head, with its gate
        pd = None if pos is not None else self.pos_dev
        if self.budget:
            # the token's row is not its position
            k3, v3 = self._heads(kc), self._heads(vc)
            row_dev = None if pos is not None else self.rows_dev
            i = self.kv_index[il]
            rot = self.ops.store(self._q_view(q), k.view(1, c.n_head_kv, hd), v.view(1, c.n_head_kv, hd), k3, v3,
                                 self.all_pos[pos:pos + 1] if pd is None else pd, self.n_rows, q_norm=qn, k_norm=kn, mode=mode,
                                 eps=c.eps, rope_dim=c.n_rot, freq_base=c.freq_base, q_out=q_rot.view(1, c.n_head, hd),
                                 row0_dev=row_dev, acc=self.kv_acc[i], row_pos=self.kv_pos[i], stream=s)
            self.ops.tree_attention(rot, k3, v3, self.n_rows, gate=self._gate_view(q), acc=self.kv_acc[i],
                                    out=att.view(1, c.n_head, hd), n_past_dev=row_dev, stream=s)
        else:
            self._store(q, k, v, q_rot, kc, vc, qn, kn, mode, hx, s, pos)
            # the split attention for blocks, and beyond the positions that the one-CTA attention takes
            if self.ops and (self.blocks or (self.max_ctx if pos is None else pos + 1) > self.plain_rows):
                args = dict(gate=self._gate_view(q), out=att.view(1, c.n_head, hd), n_past_dev=pd, stream=s)
                rot, k3, v3, n = q_rot.view(1, c.n_head, hd), self._heads(kc), self._heads(vc), pos or 0
                if self.blocks:
                    bc, bounds = self.blocks, self.bounds[self.kv_index[il]]
                    self.ops.block_attention(rot, k3, v3, bounds, n, n_sink=bc.n_sink, n_local=bc.n_local, n_sel=bc.n_sel,
                                             **args)
                    # the row just stored may complete a block
                    if pos is None:
                        self.ops.block_bounds(k3, bounds, row1_dev=pd, stream=s)
                    elif (pos + 1) % bc.block == 0:
                        self.ops.block_bounds(k3, bounds, pos, pos + 1, stream=s)
                else:
                    self.ops.tree_attention(rot, k3, v3, n, **args)
            elif c.attn_gate or c.n_rot != hd:
                n_pos = pos + 1 if pos is not None else self.max_ctx
                gate = _ptr(q) + 4 * hd if c.attn_gate else None
                _ok(hx.hoard_hx_attention_ex(_ptr(q_rot), _ptr(kc), _ptr(vc), c.n_head, c.n_head_kv, hd, n_pos, _ptr(pd),
                                             scale, gate, qs, _ptr(att), self.kv_type, s), "attention")
            elif pos is None:
                _ok(hx.hoard_hx_attention_at(_ptr(q_rot), _ptr(kc), _ptr(vc), c.n_head, c.n_head_kv, hd,
                                             _ptr(self.pos_dev), self.max_ctx, scale, _ptr(att), self.kv_type, s),
                    "attention")
            else:
                _ok(hx.hoard_hx_attention(_ptr(q_rot), _ptr(kc), _ptr(vc), c.n_head, c.n_head_kv, hd, pos + 1, scale,
                                          _ptr(att), self.kv_type, s), "attention")
        _ok(hx.hoard_hx_quant_q8(_ptr(att), self.nq, _ptr(self.q8), s), "quant")
        ty, wo = L["o"]
        _ok(hx.hoard_hx_gemv(ty, _ptr(wo), H, self.nq, _ptr(self.q8), _ptr(x), _ptr(x2), s), "gemv")

    def _store(self, q, k, v, q_rot, kc, vc, qn, kn, mode, hx, s, pos):
        """QK norm, RoPE, and k, v to the cache row of the token's position."""
        c, hd = self.cfg, self.cfg.head_dim
        if c.attn_gate or c.n_rot != hd:
            # fused q + gate rows ([q | gate] per head), partial rotary dims
            qs = 2 * hd if c.attn_gate else hd
            pd = None if pos is not None else _ptr(self.pos_dev)
            _ok(hx.hoard_hx_qknorm_rope_store_ex(_ptr(q), _ptr(k), _ptr(v), _ptr(qn), _ptr(kn), mode, c.eps, c.n_head,
                                                 c.n_head_kv, hd, qs, c.n_rot, pos if pos is not None else 0, pd,
                                                 self.max_ctx, c.freq_base, _ptr(q_rot), _ptr(kc), _ptr(vc), self.kv_type,
                                                 s), "qk rope")
        elif pos is None:
            _ok(hx.hoard_hx_qknorm_rope_store_at(_ptr(q), _ptr(k), _ptr(v), _ptr(qn), _ptr(kn), mode, c.eps, c.n_head,
                                                 c.n_head_kv, hd, _ptr(self.pos_dev), self.max_ctx, c.freq_base,
                                                 _ptr(q_rot), _ptr(kc), _ptr(vc), self.kv_type, s), "qk rope")
        else:
            _ok(hx.hoard_hx_qknorm_rope_store(_ptr(q), _ptr(k), _ptr(v), _ptr(qn), _ptr(kn), mode, c.eps, c.n_head,
                                              c.n_head_kv, hd, pos, c.freq_base, _ptr(q_rot), _ptr(kc), _ptr(vc),
                                              self.kv_type, s), "qk rope")

    def _q_view(self, q):
        """One token's q projection as [1][n_head][head_dim] (heads of a fused q + gate projection lie apart)."""
        c = self.cfg
        return q.view(1, c.n_head, -1)[:, :, :c.head_dim]

    def _gate_view(self, q):
        c = self.cfg
        return q.view(1, c.n_head, -1)[:, :, c.head_dim:] if c.attn_gate else None

    def _layer_gdn(self, il, L, x, x2, hx, s, pos=None):
        """A gated delta-net block (src/run_qwen35.cpp:508-553): x2 = W_out gdn(RMSNorm(x) * attn_norm) + x."""
        c = self.cfg
        H, r = c.n_embd, self.rec_index[il]
        _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x), H, c.eps, _ptr(L["attn_norm"]), _ptr(self.q8), s), "rmsnorm_q8")
        _ok(hx.hoard_hx_gemv_multi(3, L["qkv_types"], L["qkv_w"], self.gdn_N, H, _ptr(self.q8), None, self.gdn_y, s),
            "gemv qkv z ba")
        _ok(hx.hoard_hx_gdn_step(_ptr(self.gdn_qkv), _ptr(self.gdn_z), _ptr(self.gdn_ba), _ptr(L["conv_w"]),
                                 _ptr(self.gdn_ring[r]), _ptr(L["dt_bias"]), _ptr(L["ssm_a"]), _ptr(L["ssm_norm"]),
                                 _ptr(self.gdn_state[r]), c.ssm_dt_rank, c.ssm_n_group, c.ssm_d_state, c.ssm_d_conv,
                                 c.eps, pos if pos is not None else 0, None if pos is not None else _ptr(self.pos_dev),
                                 _ptr(self.gdn_out), s), "gdn step")
        _ok(hx.hoard_hx_quant_q8(_ptr(self.gdn_out), self.gdn_vd, _ptr(self.q8), s), "quant")
        ty, wo = L["o"]
        _ok(hx.hoard_hx_gemv(ty, _ptr(wo), H, self.gdn_vd, _ptr(self.q8), _ptr(x), _ptr(x2), s), "gemv")

    def reset_state(self):
        """Zeroes the delta-net states (the start of a sequence; src/run_qwen35.cpp:366-373) and empties a bounded
        cache."""
        self.n_rows = 0
        if hasattr(self, "gdn_state"):
            self.gdn_state.zero_()

    def _step_at(self, stream=None):
        """One decode step at the device position: token seq[pos] -> seq[pos + 1], pos += 1."""
        c, hx, s = self.cfg, _hx(), _stream(stream)
        H = c.n_embd
        x, x2 = self.x, self.x2
        _ok(hx.hoard_hx_embed_at(self.embd_type, _ptr(self.embd), H, c.n_vocab, _ptr(self.seq), _ptr(self.pos_dev),
                                 _ptr(x), s), "embed")
        for il, L in enumerate(self.layers):
            self._layer_attention(il, L, x, x2, hx, s)
            self.moe.layers(il, 1, x2.view(1, H), stream=stream)
            x, x2 = x2, x
        _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x), H, c.eps, _ptr(self.out_norm), _ptr(self.q8), s), "rmsnorm_q8")
        _ok(hx.hoard_hx_gemv(self.out_type, _ptr(self.out_w), c.n_vocab, H, _ptr(self.q8), None, _ptr(self.logits), s),
            "gemv")
        _ok(hx.hoard_hx_argmax_at(_ptr(self.logits), c.n_vocab, _ptr(self.seq), _ptr(self.pos_dev), self.seq.numel(), s),
            "argmax")
        if self.budget:
            self.rows_dev.add_(1)

    def prefill(self, prompt, stream=None):
        """Runs the prompt tokens but the last through the step (their KV entries), then sets the
        device position to the last prompt token."""
        T = len(prompt)
        self.reset_state()
        self.seq[:T].copy_(torch.tensor(prompt, dtype=torch.int32))
        for p in range(T - 1):
            self.step(p, self.scratch_tok, stream)
        self.pos_dev.fill_(T - 1)
        if self.budget:
            self.rows_dev.fill_(self.n_rows)

    def capture(self):
        """Captures one decode step (position in device memory) as a CUDA graph."""
        if self._graph is None:
            torch.cuda.synchronize(self.dev)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                self._step_at()
            self._graph = g
        return self._graph

    def generate_graphed(self, prompt, n_gen: int):
        """Greedy decode like generate(), each generated token one replay of the captured step."""
        T = len(prompt)
        if T < 1 or T + n_gen > self.max_ctx:
            raise ValueError("prompt + n_gen must fit max_ctx")
        g = self.capture()
        self.prefill(prompt)
        for i in range(n_gen):
            if self.budget and self.n_rows == self.budget.rows:
                self._make_room(T - 1 + i)
                self.rows_dev.fill_(self.n_rows)
            g.replay()
            self.n_rows += 1
        torch.cuda.synchronize(self.dev)
        self.moe.sync_status()
        return self.seq[T:T + n_gen].tolist()

    def forward_batch(self, tokens, base: int, stream=None) -> torch.Tensor:
        """One forward over m <= max_batch consecutive tokens at positions base .. base+m-1 (causal:
        token i attends to positions <= base+i; K/V stored for all m), the MoE layers batched (T = m).
        Returns the logits [m][vocab]; row i predicts position base+i+1. hoard's verify pass,
        src/run_specloop.cpp:76-150."""
        c, hx, s = self.cfg, _hx(), _stream(stream)
        m, H, hd = len(tokens), c.n_embd, c.head_dim
        if c.full_attn_interval > 0:
            raise ValueError("batched forward of a hybrid (delta-net) model is not supported: its state is sequential")
        if self.budget:
            raise ValueError("batched forward over a bounded cache is not supported: its rows are not positions")
        if not 1 <= m <= self.max_batch or base + m > self.max_ctx:
            raise ValueError("batch must be 1..max_batch tokens inside max_ctx")
        self.seq[base:base + m].copy_(torch.tensor(tokens, dtype=torch.int32))
        if not hasattr(self, "_xb"):
            z = lambda *sh: torch.zeros(*sh, dtype=torch.float32, device=self.dev)
            self._xb, self._x2b, self._curb = z(self.max_batch, H), z(self.max_batch, H), z(self.max_batch, H)
            self._qb, self._kb, self._vb = z(self.max_batch, self.nqp), z(self.max_batch, self.nkv), z(self.max_batch, self.nkv)
            self._attb, self._lgb = z(self.max_batch, self.nq), z(self.max_batch, c.n_vocab)
        xb, x2b, cur = self._xb, self._x2b, self._curb
        for i in range(m):
            _ok(hx.hoard_hx_embed(self.embd_type, _ptr(self.embd), H, c.n_vocab, _ptr(self.seq[base + i:base + i + 1]),
                                  _ptr(xb[i]), s), "embed")
        if not hasattr(self, "_qrb"):
            self._qrb = torch.zeros(self.max_batch, self.nq, dtype=torch.float32, device=self.dev)
            self._qkv_yb = [_parr([self._qb[i].data_ptr(), self._kb[i].data_ptr(), self._vb[i].data_ptr()])
                            for i in range(self.max_batch)]
        for il, L in enumerate(self.layers):
            for i in range(m):
                bufs = (self._qb[i], self._kb[i], self._vb[i], self._qrb[i], self._attb[i], self._qkv_yb[i])
                self._layer_attention(il, L, xb[i], x2b[i], hx, s, base + i, bufs)
            self.moe.layers(il, 1, x2b[:m], stream=stream)
            xb, x2b = x2b, xb
        for i in range(m):
            _ok(hx.hoard_hx_rmsnorm_q8(_ptr(xb[i]), H, c.eps, _ptr(self.out_norm), _ptr(self.q8), s), "rmsnorm_q8")
            _ok(hx.hoard_hx_gemv(self.out_type, _ptr(self.out_w), c.n_vocab, H, _ptr(self.q8), None,
                                 _ptr(self._lgb[i]), s), "gemv")
        return self._lgb[:m].clone()

    def speculative_generate(self, prompt, n_gen: int, k_draft: int = 4):
        """hoard's speculative loop (src/run_specloop.cpp:189-210): draft k tokens greedily with the same
        model routed to its top-1 expert, verify them in one batched forward with the full top-k,
        accept the matching prefix, then run the corrected token. Greedy and lossless: the result
        equals generate()'s. Returns (tokens, {"rounds", "proposed", "accepted"})."""
        T, k_full = len(prompt), self.cfg.n_expert_used
        if self.budget:
            raise ValueError("speculative decode over a bounded cache is not supported: its rows are not positions")
        if T < 1 or T + n_gen + k_draft + 1 > self.max_ctx or not 1 <= k_draft <= self.max_batch:
            raise ValueError("prompt + n_gen + k_draft must fit max_ctx, 1 <= k_draft <= max_batch")
        self.seq[:T].copy_(torch.tensor(prompt, dtype=torch.int32))
        for p in range(T):
            self.step(p, self.scratch_tok)
        pred = self.logits.clone()
        cur, out, stats = T, [], {"rounds": 0, "proposed": 0, "accepted": 0}
        while len(out) < n_gen:
            draft, lg, dpos = [], pred, cur
            self.moe.set_top_k(1)
            try:
                for _ in range(k_draft):
                    d = int(torch.argmax(lg).item())
                    draft.append(d)
                    self.seq[dpos] = d
                    self.step(dpos, self.scratch_tok)
                    lg = self.logits.clone()
                    dpos += 1
            finally:
                self.moe.set_top_k(k_full)
            V = self.forward_batch(draft, cur)
            n, last = 0, pred
            for j in range(k_draft):
                tgt_l = pred if j == 0 else V[j - 1]
                if draft[j] == int(torch.argmax(tgt_l).item()):
                    n += 1
                    if j == k_draft - 1:
                        last = V[k_draft - 1]
                else:
                    last = tgt_l
                    break
            stats["rounds"] += 1
            stats["proposed"] += k_draft
            stats["accepted"] += n
            out += draft[:n]
            cur += n
            if len(out) >= n_gen:
                break
            corrected = int(torch.argmax(last).item())
            out.append(corrected)
            self.seq[cur] = corrected
            self.step(cur, self.scratch_tok)
            pred = self.logits.clone()
            cur += 1
        self.moe.sync_status()
        return out[:n_gen], stats

    # ---- trees of drafted tokens ----
    def forward_tree(self, tokens, parents, base: int, stream=None) -> torch.Tensor:
        """One forward over a tree of m <= max_batch drafted tokens after `base` past positions: parents[i] is the
        drafted token that token i follows (an earlier index), or -1 for the last past token. Token i takes position
        base + its depth, its k and v cache row base + i; it attends to the past, its ancestors and itself. The layers'
        attention is one call for all tokens, and so are the MoE layers (T = m). Returns the logits [m][vocab]; row i
        predicts what follows token i. With parents = [-1, 0, 1, ..] it is forward_batch, but for the order of the attention's
        sums. With `blocks` every token attends the blocks that are chosen for a past of `base` rows, its ancestors and itself:
        where blocks are left out that is not forward_batch's or the step's choice, which goes by the token's own position."""
        if stream is not None:                   # the tensors made here belong to the stream that uses them
            with torch.cuda.stream(torch.cuda.ExternalStream(_stream(stream), device=self.dev)):
                return self.forward_tree(tokens, parents, base)
        c, hx, s = self.cfg, _hx(), _stream(stream)
        m, H, hd = len(tokens), c.n_embd, c.head_dim
        words, depth = cache.tree_visibility(parents)
        if c.full_attn_interval > 0:
            raise ValueError("batched forward of a hybrid (delta-net) model is not supported: its state is sequential")
        if self.budget:
            raise ValueError("batched forward over a bounded cache is not supported: its rows are not positions")
        if len(parents) != m or m > self.max_batch or base < 0 or base + m > self.max_ctx:
            raise ValueError("a tree has a parent for each of its 1..max_batch tokens, inside max_ctx")
        if self._tree_ops is None:
            self._tree_ops = cache.CacheOps(**self._ops_args, max_tokens=min(self.max_batch, self.max_ctx), max_acc_tokens=0)
            z = lambda *sh: torch.zeros(*sh, dtype=torch.float32, device=self.dev)
            B = self.max_batch
            self._tq, self._tk, self._tv = z(B, self.nqp), z(B, self.nkv), z(B, self.nkv)
            self._tx, self._tx2, self._trot, self._tatt = z(B, H), z(B, H), z(B, self.nq), z(B, self.nq)
            self._tlg = z(B, c.n_vocab)
            self._tqkv = [_parr([self._tq[i].data_ptr(), self._tk[i].data_ptr(), self._tv[i].data_ptr()]) for i in range(B)]
        self._tree_m = m
        vis = torch.tensor(words, dtype=torch.int64).to(self.dev)
        pos = torch.tensor([base + d for d in depth], dtype=torch.int32).to(self.dev)
        tok = torch.tensor(list(tokens), dtype=torch.int32).to(self.dev)
        x, x2 = self._tx, self._tx2
        for i in range(m):
            _ok(hx.hoard_hx_embed(self.embd_type, _ptr(self.embd), H, c.n_vocab, _ptr(tok[i:i + 1]), _ptr(x[i]), s), "embed")
        q = self._tq[:m].view(m, c.n_head, -1)
        mode = QK_MODE[c.qk_norm]
        for il, L in enumerate(self.layers):
            for i in range(m):
                _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x[i]), H, c.eps, _ptr(L["attn_norm"]), _ptr(self.q8), s), "rmsnorm_q8")
                _ok(hx.hoard_hx_gemv_multi(3, L["qkv_types"], L["qkv_w"], self.qkv_N, H, _ptr(self.q8), None, self._tqkv[i],
                                           s), "gemv qkv")
            j = self.kv_index[il]
            k3, v3 = self._heads(self.kc[j]), self._heads(self.vc[j])
            rot = self._tree_ops.store(q[:, :, :hd], self._tk[:m].view(m, c.n_head_kv, hd),
                                       self._tv[:m].view(m, c.n_head_kv, hd), k3, v3, pos, base, q_norm=L.get("q_norm"),
                                       k_norm=L.get("k_norm"), mode=mode, eps=c.eps, rope_dim=c.n_rot,
                                       freq_base=c.freq_base, q_out=self._trot[:m].view(m, c.n_head, hd), stream=s)
            args = dict(vis=vis, gate=q[:, :, hd:] if c.attn_gate else None, out=self._tatt[:m].view(m, c.n_head, hd), stream=s)
            if self.blocks:
                bc = self.blocks
                self._tree_ops.block_attention(rot, k3, v3, self.bounds[j], base, n_sink=bc.n_sink, n_local=bc.n_local,
                                               n_sel=bc.n_sel, **args)
            else:
                self._tree_ops.tree_attention(rot, k3, v3, base, **args)
            ty, wo = L["o"]
            for i in range(m):
                _ok(hx.hoard_hx_quant_q8(_ptr(self._tatt[i]), self.nq, _ptr(self.q8), s), "quant")
                _ok(hx.hoard_hx_gemv(ty, _ptr(wo), H, self.nq, _ptr(self.q8), _ptr(x[i]), _ptr(x2[i]), s), "gemv")
            self.moe.layers(il, 1, x2[:m], stream=stream)
            x, x2 = x2, x
        for i in range(m):
            _ok(hx.hoard_hx_rmsnorm_q8(_ptr(x[i]), H, c.eps, _ptr(self.out_norm), _ptr(self.q8), s), "rmsnorm_q8")
            _ok(hx.hoard_hx_gemv(self.out_type, _ptr(self.out_w), c.n_vocab, H, _ptr(self.q8), None, _ptr(self._tlg[i]), s),
                "gemv")
        return self._tlg[:m].clone()

    def accept(self, base: int, path, stream=None):
        """After forward_tree at `base`: the k and v of the drafted tokens path[0], path[1], .. (a root and its accepted
        descendants) become cache rows base, base + 1, .."""
        path = list(path)
        if path and (self._tree_ops is None or path[-1] >= self._tree_m):
            raise ValueError("a path names tokens of the last forward_tree")
        for j in range(len(self.kv_index)):
            k3, v3 = self._heads(self.kc[j]), self._heads(self.vc[j])
            if path:
                self._tree_ops.take(k3, v3, base, path, stream=stream)
            if self.blocks and path:
                self._tree_ops.block_bounds(k3, self.bounds[j], base, base + len(path), stream=stream)

    def tree_generate(self, prompt, n_gen: int, depth: int = 4, width: int = 2):
        """speculative_generate with a tree: at each of `depth` levels the draft (this model at its top-1 expert) offers its
        `width` best tokens and goes on from the best; one forward_tree verifies all of them, the longest path that the
        full model agrees with is accepted, then the corrected token runs. Greedy; the tokens are generate()'s wherever the
        model's best two logits differ by more than the order of f32 sums moves them (verification sums in another order).
        With `blocks` only where they hold the whole sequence (see forward_tree). Returns (tokens, {"rounds", "proposed",
        "accepted"})."""
        T, k_full = len(prompt), self.cfg.n_expert_used
        if self.budget or self.cfg.full_attn_interval > 0:
            raise ValueError("a tree of drafts needs a cache whose rows are positions, and no delta-net state")
        if (T < 1 or depth < 1 or width < 1 or depth * width > self.max_batch
                or T + n_gen + depth * width + 1 > self.max_ctx):
            raise ValueError("prompt + n_gen + the tree must fit max_ctx, depth * width <= max_batch")
        if self.blocks and self.blocks.leaves_out(T + n_gen + depth):
            raise ValueError("a tree of drafts attends the blocks chosen for the past before it: its tokens are generate()'s only "
                             "where n_sink + n_local + n_sel blocks hold the whole sequence")
        self.seq[:T].copy_(torch.tensor(prompt, dtype=torch.int32))
        self.reset_state()
        for p in range(T):
            self.step(p, self.scratch_tok)
        pred = self.logits.clone()
        cur, out, stats = T, [], {"rounds": 0, "proposed": 0, "accepted": 0}
        while len(out) < n_gen:
            tokens, parents, lg, parent = [], [], pred, -1
            self.moe.set_top_k(1)
            try:
                for d in range(depth):
                    best = torch.topk(lg, width).indices.tolist()
                    first = len(tokens)
                    tokens += best
                    parents += [parent] * width
                    parent = first
                    if d + 1 < depth:
                        self.seq[cur + d] = best[0]
                        self.step(cur + d, self.scratch_tok)
                        lg = self.logits.clone()
            finally:
                self.moe.set_top_k(k_full)
            V = self.forward_tree(tokens, parents, cur)
            path, at, want = [], -1, int(torch.argmax(pred).item())
            while True:
                hit = [i for i, (t, p) in enumerate(zip(tokens, parents)) if p == at and t == want]
                if not hit:
                    break
                at = hit[0]
                path.append(at)
                want = int(torch.argmax(V[at]).item())
            self.accept(cur, path)
            stats["rounds"] += 1
            stats["proposed"] += len(tokens)
            stats["accepted"] += len(path)
            out += [tokens[i] for i in path]
            cur += len(path)
            if len(out) >= n_gen:
                break
            out.append(want)
            self.seq[cur] = want
            self.step(cur, self.scratch_tok)
            pred = self.logits.clone()
            cur += 1
        self.moe.sync_status()
        return out[:n_gen], stats

    def score(self, tokens, first: int, stream=None) -> torch.Tensor:
        """Teacher-forced logits: runs tokens[0 .. n-2] through the decode step and returns the logits
        that predict tokens[first .. n-1] ([n - first][vocab])."""
        n = len(tokens)
        if not 1 <= first < n or n > self.max_ctx:
            raise ValueError("need 1 <= first < len(tokens) <= max_ctx")
        self.reset_state()
        self.seq[:n].copy_(torch.tensor(tokens, dtype=torch.int32))
        out = torch.empty(n - first, self.cfg.n_vocab, dtype=torch.float32, device=self.dev)
        for p in range(n - 1):
            self.step(p, self.scratch_tok, stream)
            if p >= first - 1:
                out[p - (first - 1)].copy_(self.logits)
        self.moe.sync_status(stream)
        return out

    def generate(self, prompt, n_gen: int, stop_at_eos: bool = False, logits_out: torch.Tensor | None = None,
                 stream=None):
        """Greedy decode of n_gen tokens after `prompt` (a list of ids). logits_out [n_gen][vocab], if given,
        receives the logits each generated token was chosen from. Returns the generated ids."""
        T = len(prompt)
        if T < 1 or T + n_gen > self.max_ctx:
            raise ValueError("prompt + n_gen must fit max_ctx")
        self.reset_state()
        self.seq[:T].copy_(torch.tensor(prompt, dtype=torch.int32))
        for p in range(T + n_gen - 1):
            out = self.seq[p + 1:p + 2] if p >= T - 1 else self.scratch_tok
            self.step(p, out, stream)
            if p >= T - 1 and logits_out is not None:
                logits_out[p - (T - 1)].copy_(self.logits)
            if stop_at_eos and p >= T - 1 and int(self.seq[p + 1].item()) == self.eos_id:
                return self.seq[T:p + 2].tolist()
        self.moe.sync_status(stream)
        return self.seq[T:T + n_gen].tolist()
