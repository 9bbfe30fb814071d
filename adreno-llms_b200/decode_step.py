"""The projection set of one decode step, driven through the C ABI.

Mirrors the call points of the reference's decode loop
(src/models/smollm2-135m-instruct/src/model.cpp:88-239): per layer a fused QKV
launch, o_proj + residual, fused gate/up/SiLU, down + residual, then the lm_head
GEMV and the arg-max.  The rotation, the key/value cache and the attention between
q/k/v and o_proj are part of it where `attention` is given.  Two wirings:

  fixed inputs   each projection reads a fixed N(0,1) activation buffer, as in a host
                 program whose own kernels sit between the projections; only the in-place
                 residual adds depend on one another.
  chained        the data flows as in the model: QKV and gate/up read the residual stream
                 (through the fused layer norms when norm=True), o_proj reads q (attention
                 itself is not on the path, so q stands in for its output), down reads the
                 SwiGLU output, lm_head reads the final residual stream.  Every projection
                 then waits for the one before it, which is what a decode step's latency is
                 made of.

Several copies ("sets") of the weights can be resident so that consecutive steps
stream from HBM rather than L2.
"""
import numpy as np

from . import KVBatch, QuantWeight
from . import synth


class Attention:
    """What a decode step keeps for the attention of its M sequences, one new token each: per layer a paged cache with
    random contents up to `lengths`, and one batch for all layers.  cache: "fp16", "int8" or "fp8"."""

    def __init__(self, ctx, shape, M, lengths, cache="int8", page=64, max_len=0, head_dim=64, window=0, sinks=0, rope_base=10000.0, seed=7, host=None):
        self.ctx, self.D, self.cache, self.window, self.sinks = ctx, head_dim, cache, window, sinks
        self.q_heads, self.kv_heads, self.M = shape.q_dim // head_dim, shape.kv_dim // head_dim, M
        self._one_per_row(lengths)
        self.max_len = max_len or max(lengths) + 16
        per_seq = -(-self.max_len // page)
        rng = np.random.default_rng(seed)
        self.table = rng.permutation(M * per_seq).astype(np.int32).reshape(M, per_seq)
        angle = np.arange(self.max_len)[:, None] * rope_base ** (-np.arange(0, head_dim, 2) / head_dim)
        self.cos_host, self.sin_host = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.cos, self.sin = ctx.upload(self.cos_host), ctx.upload(self.sin_host)
        self.row_start, self.kv_len, self.table_dev = ctx.upload(np.arange(M + 1, dtype=np.int32)), ctx.alloc(4 * M), ctx.upload(self.table)
        self.batch = KVBatch(M, M, 1, self.max_len, per_seq, self.row_start, self.kv_len, self.table_dev)
        self.out = ctx.alloc(M * shape.q_dim * 2)
        self.caches, self.buffers = [], []
        cells = M * per_seq * page * self.kv_heads
        starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        filled = [ctx.upload(starts), ctx.upload(np.asarray(lengths, np.int32))]
        fill = KVBatch(M, int(starts[-1]), max(1, max(lengths)), self.max_len, per_seq, *filled, self.table_dev)
        for layer in range(shape.layers):
            bufs = [ctx.alloc(cells * head_dim * (2 if cache == "fp16" else 1)) for _ in range(2)]
            bufs += [None, None] if cache == "fp16" else [ctx.alloc(cells * 2) for _ in range(2)]
            self.buffers.append(bufs)
            self.caches.append(ctx.kv_cache(cache, M * per_seq, page, self.kv_heads, head_dim, *bufs))
            if starts[-1]:
                rows = [rng.standard_normal((int(starts[-1]), shape.kv_dim)).astype(np.float16) for _ in range(2)]
                up = [ctx.upload(r.view(np.uint16)) for r in rows]
                ctx.kv_write(self.caches[-1], fill, up[0], 0, up[1], 0)
                ctx.sync()
                for b in up:
                    ctx.free(b)
                if host is not None:
                    host[f"cache.{layer}"] = rows
        for b in filled:
            ctx.free(b)
        self.set_lengths(lengths)

    def _one_per_row(self, lengths):
        if len(lengths) != self.M:
            raise ValueError(f"{len(lengths)} lengths for {self.M} sequences")

    def set_lengths(self, lengths):
        """Positions that the sequences have before the next step's token."""
        self._one_per_row(lengths)
        self.lengths = np.asarray(lengths, np.int32).copy()
        self.ctx.upload(self.lengths + 1, self.kv_len)

    def advance(self):
        self.set_lengths(self.lengths + 1)

    def enqueue(self, layer, q, k, v):
        c = self.ctx
        c.rope_kv_write(self.caches[layer], self.batch, self.cos, self.sin, self.max_len, self.D, self.q_heads, q, 0, q, 0, k, 0, v, 0)
        c.attention(self.caches[layer], self.batch, self.q_heads, q, 0, self.out, 0, self.D ** -0.5, self.window, self.sinks)

    def close(self):
        """Gives the caches and all buffers back; a recording of the step must not be launched any more."""
        for cache in self.caches:
            cache.close()
        mine = [self.cos, self.sin, self.row_start, self.kv_len, self.table_dev, self.out] if self.out else []
        for b in (*mine, *(b for bufs in self.buffers for b in bufs if b)):
            self.ctx.free(b)
        self.out, self.caches, self.buffers = None, [], []


class DecodeStep:
    def __init__(self, ctx, shape: synth.ModelShape, fmt: str, M: int = 1, n_sets: int = 1, seed: int = 1235,
                 vocab_rows=None, keep_host=False, only=None, comm=None, norm=False, gather_logits=False, chained=False, qkv_bias=False,
                 attention=None):
        self.ctx, self.shape, self.fmt, self.M = ctx, shape, fmt, M
        # with a communicator the lm_head rows are this rank's shard and the projection
        # stores into every rank's gather buffer (one buffer per weight set, so that
        # consecutive steps never share one)
        # gather_logits=False: a single-token step with the greedy pick exchanges one (value, row)
        # key per rank instead of the logits (each rank still stores its own shard of them)
        self.comm = comm
        self.gather_logits = gather_logits
        self.gathered = [comm.symm_alloc(M * shape.vocab * 2) for _ in range(n_sets)] if comm else None
        self.vocab_lo, self.vocab_n = vocab_rows if vocab_rows else (0, shape.vocab)
        rng = np.random.default_rng(seed)
        H, F = shape.hidden, shape.ffn
        self.host = {} if keep_host else None
        self.ops = [op for op in synth.decode_step_ops(shape) if only is None or op[0] == only]
        # activations (fixed inputs) and outputs
        self.x_h = self._act("x_h", M, H, rng)      # normed hidden -> QKV and gate/up
        # norm=True: the layer norms are part of the step, fused into the projections that read
        # them: QKV and gate/up take the residual stream itself through an RMSNorm prologue
        # (input_layernorm / post_attention_layernorm of the decoder layer)
        self.norm = norm
        self.chained = chained
        self.eps = 1e-5
        if norm:
            g = (1.0 + 0.1 * rng.standard_normal(H)).astype(np.float32).astype(np.float16)
            self.gamma = ctx.upload(g.view(np.uint16))
            if self.host is not None:
                self.host["gamma"] = g
        # attention: keyword arguments of Attention (at least lengths=[...], one per row); o_proj then reads its output
        if attention and not chained:
            raise ValueError("attention needs a chained step")
        self.attention = Attention(ctx, shape, M, host=self.host, **attention) if attention else None
        # qkv_bias=True: Qwen's q/k/v bias rows (src/models/qwen2-5-0-5b/src/layers/attention.cpp:413-469), one set per layer
        self.qkv_bias = None
        if qkv_bias:
            self.qkv_bias = []
            for layer in range(shape.layers):
                rows = [(0.5 * rng.standard_normal(n)).astype(np.float32).astype(np.float16) for n in (shape.q_dim, shape.kv_dim, shape.kv_dim)]
                if self.host is not None:
                    self.host[f"qkv_bias.{layer}"] = rows
                self.qkv_bias.append([ctx.upload(b.view(np.uint16)) for b in rows])
        self.x_attn = self._act("x_attn", M, shape.q_dim, rng)   # attention output -> o_proj
        self.x_act = self._act("x_act", M, F, rng)  # SwiGLU output -> down_proj
        self.resid0 = synth.activations(M, H, rng)
        self.resid = ctx.upload(self.resid0.view(np.uint16))
        self.q = ctx.alloc(M * shape.q_dim * 2)
        self.k = ctx.alloc(M * shape.kv_dim * 2)
        self.v = ctx.alloc(M * shape.kv_dim * 2)
        self.act = ctx.alloc(M * F * 2)
        self.logits = ctx.alloc(M * self.vocab_n * 2)
        self.token = ctx.alloc(4)
        # weights: one host copy, n_sets device copies
        self.sets = [dict() for _ in range(n_sets)]
        self.weight_bytes = 0
        for kind, layer, ws in self.ops:
            for j, (n, k) in enumerate(ws):
                name = f"{kind}.{layer}.{j}"
                if kind == "lm_head":
                    Wfull, sfull = synth.weight(fmt, shape.vocab, k, rng)
                    lo, cnt = self.vocab_lo, self.vocab_n
                    W = Wfull[lo:lo + cnt]
                    s = None if sfull is None else sfull[lo:lo + cnt]
                else:
                    W, s = synth.weight(fmt, n, k, rng)
                if self.host is not None:
                    self.host[name] = (W, s)
                self.weight_bytes += W.nbytes + (0 if s is None else s.nbytes)
                for st in self.sets:
                    st[name] = QuantWeight(ctx, fmt, W, s)
        self.plans = [None] * n_sets
        self.kernels_per_step = None

    def _act(self, name, m, k, rng):
        a = synth.activations(m, k, rng)
        if self.host is not None:
            self.host[name] = a
        return self.ctx.upload(a.view(np.uint16))

    def algorithmic_bytes(self):
        total = 0
        for kind, _, ws in self.ops:
            for n, k in ws:
                if kind == "lm_head":
                    n = self.vocab_n
                total += synth.linear_bytes(self.fmt, n, k, self.M)
        return total

    def enqueue(self, set_index=0, with_argmax=True):
        """Issue the step's launches on the context's stream (or into a recording)."""
        c, s, M, sh = self.ctx, self.sets[set_index], self.M, self.shape
        ch = self.chained
        x_qkv = self.resid if (ch or self.norm) else self.x_h
        x_o = self.attention.out if self.attention else self.q if ch else self.x_attn
        x_down = self.act if ch else self.x_act
        x_head = self.resid if ch else self.x_h
        for kind, layer, ws in self.ops:
            w = [s[f"{kind}.{layer}.{j}"].buf for j in range(len(ws))]
            if kind == "qkv" and self.norm and self.qkv_bias:
                bq, bk, bv = self.qkv_bias[layer]
                c.rmsnorm_linear_qkv_bias(M, sh.hidden, self.resid, self.gamma, self.eps, w[0], sh.q_dim, w[1], sh.kv_dim, w[2], sh.kv_dim,
                                          bq, bk, bv, self.q, self.k, self.v)
            elif kind == "qkv" and self.norm:
                c.rmsnorm_linear_qkv(M, sh.hidden, self.resid, self.gamma, self.eps, w[0], sh.q_dim, w[1], sh.kv_dim, w[2], sh.kv_dim,
                                     self.q, self.k, self.v)
            elif kind == "gate_up" and self.norm:
                c.rmsnorm_gate_up_silu(M, sh.ffn, sh.hidden, self.resid, self.gamma, self.eps, w[0], w[1], self.act)
            elif kind == "qkv" and self.qkv_bias:
                bq, bk, bv = self.qkv_bias[layer]
                c.linear_qkv_bias(M, sh.hidden, x_qkv, w[0], sh.q_dim, w[1], sh.kv_dim, w[2], sh.kv_dim, bq, bk, bv, self.q, self.k, self.v)
            elif kind == "qkv":
                c.linear_qkv(M, sh.hidden, x_qkv, w[0], sh.q_dim, w[1], sh.kv_dim, w[2], sh.kv_dim, self.q, self.k, self.v)
            elif kind == "o_add":
                if self.attention:
                    self.attention.enqueue(layer, self.q, self.k, self.v)
                c.linear_add(M, sh.hidden, sh.q_dim, x_o, w[0], self.resid)
            elif kind == "gate_up":
                c.fused_gate_up_silu(M, sh.ffn, sh.hidden, x_qkv, w[0], w[1], self.act)
            elif kind == "down_add":
                c.linear_add(M, sh.hidden, sh.ffn, x_down, w[0], self.resid)
            elif self.comm and with_argmax and M == 1 and not self.gather_logits:
                self.comm.linear_argmax_sharded(self.vocab_n, sh.hidden, x_head, w[0], self.logits, self.token)
            elif self.comm:
                self.comm.linear_gather(M, self.vocab_n, sh.hidden, x_head, w[0], self.gathered[set_index])
                if with_argmax and M == 1:   # [G][1][V/G] is the full logits vector
                    c.argmax(sh.vocab, self.gathered[set_index], self.token)
            elif with_argmax and M == 1:
                # lm_head and the greedy pick in one launch (the logits are still stored)
                c.linear_argmax(self.vocab_n, sh.hidden, x_head, w[0], self.logits, self.token)
            else:
                c.linear(M, self.vocab_n, sh.hidden, x_head, w[0], self.logits)

    def record(self, with_argmax=True):
        """Record one plan per weight set (the reference's recorded-queue replay)."""
        for i in range(len(self.sets)):
            before = self.ctx.launch_count()
            self.ctx.plan_begin()
            self.enqueue(i, with_argmax)
            self.plans[i] = self.ctx.plan_end()
            self.kernels_per_step = self.ctx.L.nn_plan_num_kernels(self.plans[i])
            assert self.ctx.launch_count() == before
        return self.kernels_per_step

    def resident_runs(self, set_index=0):
        return self.ctx.L.nn_plan_num_resident_runs(self.plans[set_index])

    def launch(self, set_index=0):
        self.ctx.plan_launch(self.plans[set_index])

    def reset_residual(self):
        self.ctx.upload(self.resid0.view(np.uint16), self.resid)

    def read_logits(self):
        return self.ctx.download(self.logits, (self.M, self.vocab_n), np.uint16).view(np.float16)

    def read_token(self):
        return int(self.ctx.download(self.token, (1,), np.int32)[0])
