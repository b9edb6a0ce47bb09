"""Vision transformer on lat/lon patch tokens.

Checkpoint contract (names and shapes of makani/models/networks/vit.py:29-231): `patch_embed.proj`,
`pos_embed [1, tokens, E]`, `blocks.{i}.{norm1, norm2, attn.{qkv, proj, q_norm, k_norm}, mlp.fwd.{0,3}}`, `norm`, `head`
(linear without bias); with `fin * fout > 1` the attention heads and the MLP hidden features are split over the
channel-parallel groups (makani/mpu/layers.py:352-359,453-529).

Options beyond the reference's, all off by default: `qk_norm` (queries and keys layer-normalised per head), `rotary` (queries and keys turned by
their rows and columns on the patch grid), `attn_window` (attention reaches as many tokens before and behind a patch as this many rows of patches have:
to its north the farthest row counts from its own column on eastwards, to its south up to its own column), `register_tokens` (learned tokens in front of
the grid's that stay visible from everywhere; they are tokens of the same sequence, so that with a window they see each other and the
northernmost rows, and what is further south reaches them through the layers), `dropout_generator` "counter" (masks that are never stored).

Execution: tokens stay in one [B, tokens, E] bf16 matrix.  Every projection (qkv, attention output, both MLP layers with
bias + GELU / bias epilogues, head) is a GEMM of the in-tree tensor-core engine (`ops/linear.py`); behind dropout from a
counter the two of the MLP are two products with bias in training, and around torch's own dropout they are torch's.  Attention reads the
fused projection's output where it lies (`ops/attention.py`; behind norms and rotation in one call, `ops/rotary.py`; with attention dropout in
training it is torch's `scaled_dot_product_attention`), and the second norm of a block takes the residual sum with it (`ops/norm.py`).  On CPU /
fp32 every piece is the plain torch op.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from ...ops import linear as linear_ops
from ...ops import rotary as rotary_ops
from ...parallel.layer_norm import LayerNorm, normed, operand_dtype
from ...parallel.layers import DistributedAttention, DistributedMLP, attend_normed
from ...utils import comm
from ..common.layers import MLP, DropPath, Dropout, PatchEmbed, TokenLinear, dropout_layer, watched


class Attention(nn.Module):
    """Multi-head self attention over all tokens, or those of a window; q / k may be layer-normalised per head and turned by their positions."""

    def __init__(self, dim, input_format="traditional", num_heads=8, qkv_bias=False, qk_norm=False, attn_drop_rate=0.0,
                 proj_drop_rate=0.0, norm_layer=LayerNorm, axes=None, window=None, sinks=0, dropout_generator="torch"):
        super().__init__()
        if dim % num_heads:
            raise ValueError(f"dim {dim} is not a multiple of num_heads {num_heads}")
        self.num_heads, self.head_dim = num_heads, dim // num_heads
        self.qkv = TokenLinear(dim, 3 * dim, bias=qkv_bias)
        self.proj = TokenLinear(dim, dim)
        self.q_norm = norm_layer(self.head_dim) if qk_norm else nn.Identity()
        self.k_norm = norm_layer(self.head_dim) if qk_norm else nn.Identity()
        self.attn_drop_rate = attn_drop_rate
        self.axes, self.window, self.sinks = axes, window, sinks
        self.proj_drop = dropout_layer(proj_drop_rate, dropout_generator)

    def forward(self, x, positions=None, residual=None):
        """Attention of x; with a residual, their sum, taken along with the dropout of the projection."""
        B, N, C = x.shape
        ctx = attend_normed(self.qkv(x), self.num_heads, self.q_norm, self.k_norm, self.attn_drop_rate if self.training else 0.0, positions, self.axes,
                            self.window, self.sinks)
        y = self.proj(ctx.reshape(B, N, C))
        return self.proj_drop(y) if residual is None else self.proj_drop.add(y, residual)


class Block(nn.Module):
    """x + attn(norm1(x)), then z = norm2(.), z + mlp(z) (the second residual starts after the norm, as upstream)."""

    def __init__(self, dim, num_heads, mlp_ratio=4.0, qkv_bias=False, mlp_drop_rate=0.0, attn_drop_rate=0.0,
                 path_drop_rate=0.0, act_layer=nn.GELU, norm_layer=LayerNorm, comm_inp_name="fin", comm_hidden_name="fout", qk_norm=False, axes=None,
                 window=None, sinks=0, dropout_generator="torch"):
        super().__init__()
        sees = dict(qk_norm=qk_norm, axes=axes, window=window, sinks=sinks, dropout_generator=dropout_generator)
        hidden = int(dim * mlp_ratio)
        self.norm1, self.norm2 = norm_layer(dim), norm_layer(dim)
        self.channel_parallel = comm.get_size(comm_inp_name) * comm.get_size(comm_hidden_name) > 1
        if self.channel_parallel:
            self.attn = DistributedAttention(dim, input_format="traditional", comm_inp_name=comm_inp_name,
                                             comm_hidden_name=comm_hidden_name, num_heads=num_heads, qkv_bias=qkv_bias,
                                             attn_drop_rate=attn_drop_rate, proj_drop_rate=mlp_drop_rate, norm_layer=LayerNorm if qk_norm else None, **sees)
            self.mlp = DistributedMLP(in_features=dim, hidden_features=hidden, out_features=dim, act_layer=act_layer,
                                      drop_rate=mlp_drop_rate, input_format="traditional", comm_inp_name=comm_inp_name,
                                      comm_hidden_name=comm_hidden_name, dropout_generator=dropout_generator)
        else:
            self.attn = Attention(dim, num_heads=num_heads, qkv_bias=qkv_bias, attn_drop_rate=attn_drop_rate,
                                  proj_drop_rate=mlp_drop_rate, norm_layer=norm_layer, **sees)
            self.mlp = MLP(in_features=dim, hidden_features=hidden, out_features=dim, act_layer=act_layer, drop_rate=mlp_drop_rate,
                           input_format="traditional", dropout_generator=dropout_generator)      # fused token MLP (ops/linear.py)
        self.drop_path = DropPath(path_drop_rate) if path_drop_rate > 0.0 else nn.Identity()

    def _joint(self) -> bool:
        """Whether attention and MLP may hand on their sums with what they are added to: there is a dropout that takes it along, and nobody has to see either's own
        result."""
        return (self.training and not self.channel_parallel and isinstance(self.attn.proj_drop, Dropout) and self.attn.proj_drop.joins()
                and not (watched(self.attn, Attention.forward) or watched(self.mlp, MLP.forward) or watched(self.drop_path, nn.Identity.forward)))

    def forward(self, x, positions=None):
        # (the products' type where they run on the engine; the channel-parallel layers take what torch's norm would hand on)
        y = self.norm1(x) if self.channel_parallel else normed(self.norm1, x, operand_dtype(x))
        more = {} if positions is None else dict(positions=positions)
        if self._joint():
            # dropouts take the residual sums with them
            z = self.norm2(self.attn(y, residual=x, **more))
            return self.mlp(z.to(operand_dtype(z)), residual=z)
        a = self.drop_path(self.attn(y, **more))
        z = self.norm2.after_sum(x, a)[1] if isinstance(self.norm2, LayerNorm) else self.norm2(x + a)
        return z + self.drop_path(self.mlp(z if self.channel_parallel else z.to(operand_dtype(z))))


class VisionTransformer(nn.Module):
    def __init__(self, inp_shape=(224, 224), patch_size=(16, 16), inp_chans=3, out_chans=3, embed_dim=768, depth=12,
                 num_heads=12, mlp_ratio=4.0, qkv_bias=True, mlp_drop_rate=0.0, attn_drop_rate=0.0, path_drop_rate=0.0,
                 norm_layer="layer_norm", comm_inp_name="fin", comm_hidden_name="fout", qk_norm=False, rotary=False, rotary_base=100.0,
                 attn_window=None, register_tokens=0, dropout_generator="torch", **kwargs):
        super().__init__()
        if norm_layer != "layer_norm":
            raise NotImplementedError(f"normalization layer type {norm_layer} not implemented for ViT")
        self.img_size, self.patch_size = tuple(inp_shape), tuple(patch_size)
        self.embed_dim = self.num_features = embed_dim
        self.out_ch = out_chans
        self.comm_inp_name, self.comm_hidden_name = comm_inp_name, comm_hidden_name
        self.patch_embed = PatchEmbed(img_size=self.img_size, patch_size=self.patch_size, in_chans=inp_chans, embed_dim=embed_dim)
        self.grid = tuple(self.patch_embed.red_img_size)                       # tokens along latitude / longitude
        self.pos_embed = nn.Parameter(torch.zeros(1, self.patch_embed.num_patches, embed_dim))
        self.pos_embed.is_shared_mp = []
        self.register_tokens = register_tokens
        if register_tokens:
            self.registers = nn.Parameter(torch.zeros(1, register_tokens, embed_dim))
            self.registers.is_shared_mp = []
        axes = None
        if rotary:      # the first half of a head's channels by rows, the second by columns (registers stand at the origin)
            band = embed_dim // num_heads // 4 * 2
            if band == 0:
                raise ValueError(f"heads of {embed_dim // num_heads} channels are too narrow to be turned by rows and columns")
            axes = rotary_ops.RotaryAxes((band, band), base=rotary_base)
            self.register_buffer("token_positions", rotary_ops.grid_positions(*self.grid, first=register_tokens), persistent=False)
        if attn_window is not None and (isinstance(attn_window, bool) or not isinstance(attn_window, int) or attn_window < 0):
            raise ValueError(f"attn_window is a number of rows of patches, got {attn_window!r}")
        sees = dict(qk_norm=qk_norm, axes=axes, window=None if attn_window is None else attn_window * self.grid[1], sinks=register_tokens)
        self.pos_drop = Dropout(path_drop_rate) if dropout_generator == "counter" else nn.Dropout(p=path_drop_rate)
        rates = torch.linspace(0, path_drop_rate, depth).tolist()
        self.blocks = nn.ModuleList([
            Block(embed_dim, num_heads, mlp_ratio=mlp_ratio, qkv_bias=qkv_bias, mlp_drop_rate=mlp_drop_rate,
                  attn_drop_rate=attn_drop_rate, path_drop_rate=rates[i], norm_layer=LayerNorm,
                  comm_inp_name=comm_inp_name, comm_hidden_name=comm_hidden_name, dropout_generator=dropout_generator, **sees)
            for i in range(depth)])
        self.norm = LayerNorm(embed_dim)
        self.out_size = out_chans * self.patch_size[0] * self.patch_size[1]
        self.head = TokenLinear(embed_dim, self.out_size, bias=False)
        nn.init.trunc_normal_(self.pos_embed, std=0.02)
        if register_tokens:
            nn.init.trunc_normal_(self.registers, std=0.02)
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.trunc_normal_(m.weight, std=0.02)
                if m.bias is not None:
                    nn.init.zeros_(m.bias)
            elif isinstance(m, nn.LayerNorm):
                nn.init.ones_(m.weight)
                nn.init.zeros_(m.bias)

    def prepare_tokens(self, x):
        tokens = self.patch_embed(x).transpose(1, 2)                            # [B, tokens, E]
        tokens = tokens + self.pos_embed.to(tokens.dtype)
        if self.register_tokens:
            tokens = torch.cat([self.registers.to(tokens.dtype).expand(tokens.shape[0], -1, -1), tokens], 1)
        return self.pos_drop(tokens)

    def forward_head(self, tokens):
        B = tokens.shape[0]
        (h, w), (p, q) = self.grid, self.patch_size
        y = self.head(tokens)                                                   # [B, h*w, p*q*out]
        # token (i, j), feature (a, b, c) -> pixel (i*p + a, j*q + b) of channel c
        y = y.view(B, h, w, p, q, self.out_ch).permute(0, 5, 1, 3, 2, 4)
        return y.reshape(B, self.out_ch, h * p, w * q)

    def forward(self, x):
        tokens = self.prepare_tokens(x)
        positions = getattr(self, "token_positions", None)
        for blk in self.blocks:
            tokens = blk(tokens) if positions is None else blk(tokens, positions)
        return self.forward_head(normed(self.norm, tokens[:, self.register_tokens:] if self.register_tokens else tokens, operand_dtype(tokens)))
