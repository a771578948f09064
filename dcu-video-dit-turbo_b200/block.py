"""One DiT transformer block on the B200 kernels (benchmark configuration 4/5).

adaLN modulation -> INT8 QKV GEMM -> per-head QK RMSNorm + 3-D RoPE -> bf16 flash
attention -> INT8 out-proj -> gated residual -> adaLN -> SwiGLU FFN (INT8 fc1,
swiglu-quant, INT8 fc2) -> gated residual, on a token shard [L, C].  By default swiglu-quant
is split across the two kernels around it (SwiGLU in fc1's epilogue, the quantizer as its own
pass over the half-width product); `fuse_swiglu=False` runs the reference's operator sequence.

The reference project has no source for the block itself (it lives in the host
application's model file); only its operator set comes from the reference.  The
glue conventions (LayerNorm without affine, RMSNorm weight per head channel,
rotary on adjacent pairs with three axis bands, bf16 gate vectors) are this
package's own.  Ten kernel launches per block on one GPU (both gated residuals run in
the epilogue of the GEMM that produces their operand).
"""
from __future__ import annotations

import torch

from . import ops
from .ulysses import UlyssesSP


def make_block_params(hidden: int = 3072, heads: int = 24, head_dim: int = 128, ffn: int = 8192,
                      seed: int = 0, device="cuda", weights: str = "int8") -> dict:
    """Random-init block: weights ~N(0,0.02) quantised per output channel (symmetric
    int8, scale = absmax/127, round half even, clamp +-127), biases ~N(0,0.01),
    modulation vectors ~N(0,0.1), norm weights 1 + N(0,0.02).  `weights="mxfp4"` quantises the
    same weights (rounded to bf16) to MXFP4 on the device instead: "w4_*" and "s4_*"."""
    if weights not in ("int8", "mxfp4"):
        raise ValueError(f"weights must be int8 or mxfp4, got {weights!r}")
    g = torch.Generator(device="cpu").manual_seed(seed)
    p = {}

    def qweight(name, n, k):
        w = (torch.randn((n, k), generator=g) * 0.02)
        if weights == "mxfp4":
            p["w4_" + name], p["s4_" + name] = ops.quantize_mxfp4(w.to(torch.bfloat16).to(device))
            p["b_" + name] = (torch.randn((n,), generator=g) * 0.01).to(torch.bfloat16).to(device)
            return
        scale = (w.abs().amax(-1) / 127.0).clamp(min=1e-30)
        p["wq_" + name] = (w / scale[:, None]).round().clamp(-127, 127).to(torch.int8).to(device)
        p["ws_" + name] = scale.float().to(device)
        p["b_" + name] = (torch.randn((n,), generator=g) * 0.01).to(torch.bfloat16).to(device)

    qweight("qkv", 3 * hidden, hidden)
    qweight("out", hidden, hidden)
    qweight("fc1", 2 * ffn, hidden)
    qweight("fc2", hidden, ffn)
    for name in ("shift1", "scale1", "gate1", "shift2", "scale2", "gate2"):
        p[name] = (torch.randn((hidden,), generator=g) * 0.1).to(torch.bfloat16).to(device)
    for name in ("q_norm_w", "k_norm_w"):
        p[name] = (1.0 + torch.randn((head_dim,), generator=g) * 0.02).to(torch.bfloat16).to(device)
    p["heads"], p["head_dim"], p["hidden"], p["ffn"] = heads, head_dim, hidden, ffn
    return p


def rope_tables(positions: torch.Tensor, head_dim: int = 128, axes=(32, 48, 48),
                theta: float = 10000.0):
    """cos/sin fp32 [S, head_dim/2] for integer positions [S,3] (t, y, x): the head
    dimension is split into three axis bands; band a rotates adjacent pairs with
    frequencies theta^(-2i/band).  Computed in float64 on the host side."""
    assert sum(axes) == head_dim
    cos, sin = [], []
    pos = positions.detach().cpu().double()
    for a, band in enumerate(axes):
        half = band // 2
        inv = theta ** (-torch.arange(half, dtype=torch.float64) * 2.0 / band)
        ang = pos[:, a][:, None] * inv[None, :]
        cos.append(torch.cos(ang).float())
        sin.append(torch.sin(ang).float())
    return torch.cat(cos, -1).contiguous(), torch.cat(sin, -1).contiguous()


def grid_positions(tokens: int, height: int = 22, width: int = 38) -> torch.Tensor:
    """Synthetic (t, y, x) coordinates for a joint token stream of `tokens` rows."""
    idx = torch.arange(tokens)
    return torch.stack((idx // (height * width), (idx // width) % height, idx % width), dim=-1)


class DiTBlock:
    """`window=(left, right)` and `sinks` restrict attention to a sliding window of token positions
    and the first tokens (`ops.window_fwd_bhsd`; None: full attention).  Parameters with MXFP4
    weights (`make_block_params(weights="mxfp4")`) run the four linears in that format, on one GPU; their
    gated residual is a kernel of its own and SwiGLU part of the second projection's quantiser, so
    the attributes `fuse_residual` and `fuse_swiglu` are then False whatever was asked for."""

    def __init__(self, params: dict, sp: UlyssesSP | None = None, head_chunks: int = 1,
                 overlap: bool = True, fuse_residual: bool = True, fuse_swiglu: bool = True,
                 window: tuple[int, int] | None = None, sinks: int = 0):
        self.p = params
        self.window, self.sinks = window, sinks
        if window is None and sinks:
            raise ValueError("sinks need a window")
        self.mxfp4 = "w4_qkv" in params
        if self.mxfp4 and sp is not None and sp.world > 1:
            raise ValueError("MXFP4 weights run on one GPU: the sequence-parallel ends quantise to int8")
        # gated residual in the int8 GEMM's epilogue where it pays (same bits either way)
        self.fuse_residual = bool(fuse_residual) and not self.mxfp4
        # SwiGLU in fc1's epilogue (same bits either way): the [L, 2*ffn] projection never reaches
        # memory; needs fc1's rows interleaved gate/up in groups of 64, prepared once here
        self.fuse_swiglu = bool(fuse_swiglu) and not self.mxfp4 and params["ffn"] % ops.SWIGLU_GROUP == 0
        self._fc1_interleaved = None
        if self.fuse_swiglu:
            self._fc1_interleaved = tuple(ops.interleave_gate_up(params[k]) for k in ("wq_fc1", "ws_fc1", "b_fc1"))
        self.sp = sp
        self.head_chunks = head_chunks
        self.overlap = overlap
        self.heads = params["heads"]
        self.head_dim = params["head_dim"]

    def _attn(self, q, k, v):
        if self.window is not None:
            return ops.window_fwd_bhsd(q, k, v, self.head_dim ** -0.5, *self.window, self.sinks)
        return ops.fwd_bhsd(q, k, v, self.head_dim ** -0.5)

    def attention(self, qkv: torch.Tensor) -> torch.Tensor:
        """qkv [L,3,H,D] (normed + rotated) -> [L, H*D]."""
        L = qkv.shape[0]
        if self.sp is None or self.sp.world == 1:
            q, k, v = (qkv[:, i].transpose(0, 1).unsqueeze(0) for i in range(3))
            out = self._attn(q, k, v)              # [1,H,L,D] view of [1,L,H,D]
            return out.transpose(1, 2).reshape(L, self.heads * self.head_dim)
        o = self.sp.attention_fused(qkv, self._attn, chunks=self.head_chunks, overlap=self.overlap)
        return o.reshape(L, self.heads * self.head_dim)

    def _linear_residual(self, x, gate, q8, s, wq, ws, bias) -> None:
        """x += gate * linear(q8): one kernel (the gated residual runs in the GEMM's epilogue, so
        the linear's output never makes a round trip through memory), or, with
        `fuse_residual=False`, GEMM + gate-residual kernel; same bits either way.  Measured at
        109099 tokens on one box in alternation: out-projection (K = 3072) 1.01 ms fused against
        0.80 + 0.34 ms, fc2 (K = 8192) 2.12 against 1.95-1.99 + 0.34 ms."""
        if self.fuse_residual:
            ops.int8_gemm_dequant_residual_(x, gate, q8, s.view(-1), wq, ws, bias)
        else:
            ops.gate_residual_(x, ops.int8_gemm_dequant(q8, s.view(-1), wq, ws, bias), gate)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                taps: dict | None = None) -> torch.Tensor:
        """x bf16 [L, C] (this rank's tokens); cos/sin fp32 [L, 64] for the same rows.
        Returns a new tensor.  `taps`, when given, receives intermediate tensors for parity
        checks: "attn" = the attention output rows [L, H*D] that feed the out-projection and,
        on the single-GPU path, "qkv" = the normed and rotated projections [L,3,H,D]."""
        p = self.p
        L = x.shape[0]
        x = x.clone()
        if self.mxfp4:
            return self._forward_mxfp4(x, cos, sin, taps)
        q8, s = ops.layernorm_mod_quant(x, p["scale1"], p["shift1"])
        qkv = ops.int8_gemm_dequant(q8, s.view(-1), p["wq_qkv"], p["ws_qkv"], p["b_qkv"])
        qkv = qkv.view(L, 3, self.heads, self.head_dim)
        if self.sp is not None and self.sp.world > 1:
            # sequence parallel: norm + rotary write the all-to-all send buffer directly and
            # the out-projection's quantizer reads the reverse all-to-all's buffer in place
            if self.sp.peer is not None:
                # the kernels carry the exchange: stores into the owner ranks' buffers
                gathered = self.sp.attention_peer(
                    lambda table, row0, seq: ops.qk_norm_rope_scatter(
                        qkv, p["q_norm_w"], p["k_norm_w"], cos, sin, table, self.sp.world, row0, seq),
                    self._attn)
            else:
                send = ops.qk_norm_rope_pack(qkv, p["q_norm_w"], p["k_norm_w"], cos, sin,
                                             self.sp.world, self.head_chunks)
                gathered = self.sp.attention_packed(send, self._attn, overlap=self.overlap)
            if taps is not None:
                taps["attn"] = UlyssesSP.unpack_gathered(gathered).contiguous()
            q8, s = ops.quantize_int8_rowwise_gathered(gathered)
        else:
            ops.qk_norm_rope_(qkv, p["q_norm_w"], p["k_norm_w"], cos, sin)
            attn_rows = self.attention(qkv)
            if taps is not None:
                taps["qkv"], taps["attn"] = qkv, attn_rows
            q8, s = ops.quantize_int8_rowwise(attn_rows)
        self._linear_residual(x, p["gate1"], q8, s, p["wq_out"], p["ws_out"], p["b_out"])
        q8, s = ops.layernorm_mod_quant(x, p["scale2"], p["shift2"])
        if self.fuse_swiglu:
            h = ops.int8_gemm_dequant_swiglu(q8, s.view(-1), *self._fc1_interleaved)
            q8, s = ops.quantize_int8_rowwise(h)
        else:
            f = ops.int8_gemm_dequant(q8, s.view(-1), p["wq_fc1"], p["ws_fc1"], p["b_fc1"])
            q8, s = ops.swiglu_quantize_int8_rowwise(f)
        self._linear_residual(x, p["gate2"], q8, s, p["wq_fc2"], p["ws_fc2"], p["b_fc2"])
        return x


    def _forward_mxfp4(self, x, cos, sin, taps):
        """The same block with MXFP4 linears: every linear quantises its own input, the second FFN
        projection's with SwiGLU in front."""
        p = self.p
        linear = lambda t, name, act=None: ops.mxfp4_linear(t, p["w4_" + name], p["s4_" + name], p["b_" + name], act)  # noqa: E731
        qkv = linear(ops.layernorm_mod(x, p["scale1"], p["shift1"]), "qkv").view(x.shape[0], 3, self.heads, self.head_dim)
        ops.qk_norm_rope_(qkv, p["q_norm_w"], p["k_norm_w"], cos, sin)
        attn_rows = self.attention(qkv)
        if taps is not None:
            taps["qkv"], taps["attn"] = qkv, attn_rows
        ops.gate_residual_(x, linear(attn_rows, "out"), p["gate1"])
        f = linear(ops.layernorm_mod(x, p["scale2"], p["shift2"]), "fc1")
        return ops.gate_residual_(x, linear(f, "fc2", "swiglu"), p["gate2"])


class GraphedBlock:
    """One block pass captured in a CUDA graph (single GPU, fixed token count).

    The ten kernel launches of a pass replay as one graph launch, which removes the
    host-side launch gaps between them.  Shapes, weights and the rotary tables are
    fixed at capture time; `__call__` copies the input into the captured buffer, replays
    and returns the captured output buffer (overwritten by the next call).
    Warm-up passes run first so that one-time host work (function attributes, lookup
    tables, library loading) never happens inside the capture.
    The sequence-parallel pass stays eager: a capture that included its all-to-all
    collectives on the side stream did not come back within five minutes on two GPUs (at
    23638 and at 5910 tokens).  With the peer-store exchange the host enqueues such a pass in
    about 0.4 ms, well under the GPU time of the smallest benchmark shape."""

    def __init__(self, block: DiTBlock, x_example: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                 warmup: int = 3):
        if block.sp is not None and block.sp.world > 1:
            raise RuntimeError("GraphedBlock captures the single-GPU pass only")
        self.block = block
        self.static_x = x_example.clone()
        self.cos, self.sin = cos, sin
        side = torch.cuda.Stream(device=x_example.device)
        side.wait_stream(torch.cuda.current_stream(x_example.device))
        with torch.cuda.stream(side):
            for _ in range(warmup):
                block.forward(self.static_x, cos, sin)
        torch.cuda.current_stream(x_example.device).wait_stream(side)
        before = ops.launch_count
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.static_y = block.forward(self.static_x, cos, sin)
        self.launches_per_replay = ops.launch_count - before

    def replay(self) -> torch.Tensor:
        """Replay on whatever `static_x` currently holds; returns the captured output buffer."""
        self.graph.replay()
        ops.launch_count += self.launches_per_replay
        return self.static_y

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        self.static_x.copy_(x, non_blocking=True)
        return self.replay()
