"""Grouped softmax attention with biased projections, per-head query and key norms, a rotation over part of a head,
keys seen within a chunk or a window, and a gate on the heads' outputs.

    q, k, v = Wq x + bq, Wk x + bk, Wv x + bv          heads x dim, kv_heads x dim, kv_heads x vdim
    q <- rms(q over each head's dim) * wq;  k likewise   one weight [dim] for all heads, before the rotation
    dimensions i and i + turned/2 (i < turned/2) of every head of q and k turned by position * base^(-2i/turned)
    query at position p sees key at j <= p where   chunk c: floor(p / c) = floor(j / c);   window w: p - j < w;   else all
    softmax of q.k * scale; query head h reads key/value head h // (heads / kv_heads)
    out = Wo (heads * sigmoid(Wg x))

Variants, each a constructor parameter: `values_are_keys` (no Wv: a value is the head's own key as projected, before norm and
rotation; then vdim = dim); `head_norm_weights=False` (queries and keys over their root mean square, no weight; a turn keeps a
head's length, so such a norm ahead of the rotation and one behind it are one computation); `sink` (every softmax sum holds
one more term exp(sink), the same for all heads, with neither key nor value); `gate="head"` (one gate a head, Wg x has
`heads` numbers); `softcap` (scores become softcap * tanh(score / softcap)); `slopes` (one number a head: slope * (i - j) is taken
off the score of a query at i and a key at j); `q_temp` = (coef, every) (a query at position p is multiplied by 1 + coef
ln(floor((p + 1) / every) + 1)); `borrows` (no Wk and Wv: the keys and values are another layer's, read from the cache entry that layer
writes); `out_scale` (a factor on the mixer's output, applied to the attended heads before they are rounded); `kept` (how many of
the last positions the cache entry keeps where other layers that read it see further back than this one; 0 all of them).

The four projections are one stacked product [q | k | v | g]; the biases are added, the heads normed and turned, and
keys and values written into the pages by one kernel (`head_norm_rope_write`); the attention kernels apply a gate a head
themselves where their heads are the values' own size.  In a decode step, rows without biases whose heads turn in neighbouring
pairs (or not at all) and need no padding go through one launch instead (`attention_decode_pairs`: norm, turn, cache write,
attention, sink and gates), the cosines and sines of the step's rows made once for all layers that turn alike.  Keys have `dim` dimensions a head and
values `vdim`; both are cached as heads of one padded size (zeros beyond), which the paged attention kernels take as it
is.  Chunks are counted from a sequence's position 0, so what a row sees does not depend on how a prompt was cut; the
cache keeps a chunk's (or a window's) span of positions and gives older pages back.  Norm statistics, angles and the
softmax are float32.  Every size and constant is a constructor parameter; each mechanism can be switched off: without
`gate` there is no Wg and the heads go to Wo as they are; `rotation` (a `RotaryFrequencies`) replaces `turned` and `base`
where the frequencies are not the plain powers of the base; `neighbours` pairs dimensions 2i and 2i + 1.
"""

from __future__ import annotations

import torch

from ..weights.binder import TensorSpec
from .base import MIXERS, CacheNeed
from .conv_attention import padded_head
from .linear import Linear
from .rope import RotaryFrequencies


class GatedAttention:
    graph_safe = True
    graph_safe_rows = None
    writes_fresh = True    # forward(..., fresh=True) writes its result instead of adding it

    def __init__(self, hidden: int, n_heads: int, n_kv_heads: int, dim: int, vdim: int, scale: float, prefix: str, *,
                 bias: bool = True, head_norm_eps: float | None = None, turned: int = 0, base: float = 10000.0,
                 chunk: int = 0, window: int = 0, gate=True, rotation: RotaryFrequencies | None = None,
                 neighbours: bool = False, values_are_keys: bool = False, head_norm_weights: bool = True,
                 sink: float | None = None, softcap: float = 0.0, slopes=None, q_temp=None, borrows: bool = False,
                 out_scale: float = 1.0, kept: int | None = None):
        """`head_norm_eps` None: no query and key norms; `turned` 0: no rotation; `chunk` and `window` 0: every earlier key;
        `gate` one a value (True), one a head ("head") or none (False); `sink` None: nothing beside the keys in a sum."""
        if n_heads % n_kv_heads:
            raise ValueError(f"{n_heads} query heads do not group evenly into {n_kv_heads} kv heads")
        if chunk and window:
            raise ValueError("keys are seen by chunk or by window, not both")
        if rotation is not None:
            turned = rotation.dims
        if turned % 2 or turned > dim:
            raise ValueError(f"the rotation turns pairs of a head's {dim} dimensions, got {turned}")
        if gate not in (False, True, "head"):
            raise ValueError(f"a gate is absent, one a value (True) or one a head ('head'), got {gate!r}")
        if values_are_keys and (vdim != dim or bias):
            raise ValueError(f"values that are their keys have the keys' size {dim} (got {vdim}) and no bias")
        if softcap < 0.0 or (slopes is not None and len(slopes) != n_heads) or (q_temp is not None and int(q_temp[1]) < 1):
            raise ValueError(f"a cap on scores is not negative ({softcap}), slopes are one a head, a temperature's step is positive ({q_temp})")
        if borrows and (bias or values_are_keys or head_norm_eps is not None):
            raise ValueError("a layer that reads another layer's keys and values has queries without biases and norms")
        if rotation is not None and rotation.magnitude != 1.0 and head_norm_eps is not None and not head_norm_weights:
            raise ValueError("a rotation that changes lengths does not go with heads of unit root mean square")
        self.hidden, self.n_heads, self.n_kv_heads, self.dim, self.vdim = int(hidden), int(n_heads), int(n_kv_heads), int(dim), int(vdim)
        self.scale, self.prefix, self.bias, self.head_norm_eps = float(scale), prefix, bool(bias), head_norm_eps
        self.turned, self.chunk, self.window = int(turned), int(chunk), int(window)
        self.q_width, self.k_width, self.v_width = self.n_heads * self.dim, self.n_kv_heads * self.dim, self.n_kv_heads * self.vdim
        self.values_are_keys, self.head_norm_weights = bool(values_are_keys), bool(head_norm_weights) and head_norm_eps is not None
        self.borrows, self.softcap, self.q_temp, self.out_scale = bool(borrows), float(softcap), q_temp, float(out_scale)
        self.slope_values = [float(slope) for slope in slopes] if slopes is not None else None
        self.kept = (self.chunk or self.window) if kept is None else int(kept)
        self.qkv_width = self.q_width + (0 if self.borrows else self.k_width + (0 if self.values_are_keys else self.v_width))
        self.gate_width = self.n_heads * self.vdim
        self.gate_per_head = gate == "head"
        self.sink = None if sink is None else float(sink)
        self.pad = padded_head(dim, vdim)
        self.gate, self.neighbours = bool(gate), bool(neighbours)
        self.rotation = rotation if rotation is not None else (RotaryFrequencies(self.turned, base) if self.turned else None)
        slices = [(self.q_width, "q")]
        if not self.borrows:
            slices += [(self.k_width, "k")] + ([] if self.values_are_keys else [(self.v_width, "v")])
        if self.gate:
            slices.append((self.n_heads if self.gate_per_head else self.gate_width, "g"))
        self.proj = Linear(hidden, [width for width, _ in slices], [prefix + name for _, name in slices], whole=16 if self.gate_per_head else 1)
        self.out = Linear(self.gate_width, hidden, prefix + "o")
        self.q_norm = self.k_norm = self.qkv_bias = self.sinks = self.slopes = None

    def keep_in_float8(self):
        self.proj.keep_in_float8()
        self.out.keep_in_float8()

    @property
    def input_reader(self):
        return self.proj.reader()

    def tensor_specs(self):
        specs = self.proj.tensor_specs() + self.out.tensor_specs()
        if self.bias:
            specs += [TensorSpec(self.prefix + "q.b", (self.q_width,), "linear"), TensorSpec(self.prefix + "k.b", (self.k_width,), "linear"),
                      TensorSpec(self.prefix + "v.b", (self.v_width,), "linear")]
        if self.head_norm_weights:
            specs += [TensorSpec(self.prefix + "q.norm", (self.dim,), "norm"), TensorSpec(self.prefix + "k.norm", (self.dim,), "norm")]
        return specs

    def load(self, get):
        self.proj.load(get)
        self.out.load(get)
        if self.bias:
            self.qkv_bias = torch.cat([get(self.prefix + name).to(torch.float32) for name in ("q.b", "k.b", "v.b")]).contiguous()
        if self.sink is not None:
            self.sinks = torch.full((self.n_heads,), self.sink, dtype=torch.float32, device=self.proj.weight.device)
        if self.slope_values is not None:
            self.slopes = torch.tensor(self.slope_values, dtype=torch.float32, device=self.out.weight.device)
        if self.head_norm_weights:
            self.q_norm = get(self.prefix + "q.norm").to(torch.float32).contiguous()
            self.k_norm = get(self.prefix + "k.norm").to(torch.float32).contiguous()

    def prepare(self, kernels):
        self.proj.prepare(kernels)
        self.out.prepare(kernels)

    def cache_need(self):
        # a chunk is at most `chunk` positions long: nothing older than that is ever seen again
        return CacheNeed(kind="kv", kv_heads=self.n_kv_heads, head_dim=self.pad, window=self.kept)

    def working_bytes(self, step) -> int:
        total = self.proj.working_bytes(step, step.rows) + 2 * step.matrix(step.rows, self.n_heads * self.pad)
        total += step.matrix(step.rows, self.gate_width, reader=self.out.reader_for_plan(step.act_size))
        if self.rotation is not None and step.rows <= step.seqs:      # a decode step's cosines and sines
            total += 2 * step.matrix(step.rows, self.turned // 2, 4)
        if step.sizes is not None:
            total += step.sizes.attention_working_bytes(step.rows, step.seqs, step.max_rows_per_seq, self.n_heads, self.n_kv_heads,
                                                        self.pad, step.max_position, step.act_size, window=self.window, chunk=self.chunk)
        return total + self.out.working_bytes(step, step.rows, accumulate=True)

    def forward(self, ctx, x, hidden, cache, then_norm=None, fresh=False):
        k = ctx.kernels
        n = ctx.n_rows
        proj = self.proj.forward(ctx, x)
        no_padding = self.pad == self.dim == self.vdim
        # the attended heads are the output projection's input as they leave the attention kernel
        plain = self.pad == self.vdim and (not self.gate or self.gate_per_head)
        ending = dict(sinks=self.sinks) if self.sinks is not None else {}
        if plain and self.gate_per_head:
            ending.update(gates=proj, gate_first=self.qkv_width)
        if self.softcap:
            ending["softcap"] = self.softcap
        if self.slopes is not None:
            ending["slopes"] = self.slopes
        if self.q_temp is not None:
            ending["q_temp"] = self.q_temp
        if self.out_scale != 1.0:
            ending["out_scale"] = self.out_scale
        in_one = getattr(k, "attention_decode_pairs", None)
        if (in_one is not None and ctx.is_decode and plain and no_padding and self.qkv_bias is None and (self.neighbours or self.rotation is None)
                and k.attention_decode_pairs_takes(proj.dtype, self.pad, self.n_heads, self.n_kv_heads)):
            cos, sin = self.rotation.row_angles(ctx) if self.rotation is not None else (None, None)
            attended = ctx.new_activations(n, self.gate_width, reader=self.out.reader())
            if in_one(proj, 0, attended, self.q_norm, self.k_norm, self.head_norm_eps or 0.0, cos, sin, ctx.positions, cache.k_pages, cache.v_pages,
                      cache.page_table, self.n_heads, self.n_kv_heads, self.pad, self.scale, cache.writes, ctx, window=self.window, chunk=self.chunk,
                      unit_norm=self.head_norm_eps is not None and not self.head_norm_weights, values_are_keys=self.values_are_keys, **ending):
                self.out.forward(ctx, attended, out=hidden, accumulate=not fresh)
                return None
        q = self._queries(ctx, proj, cache)
        attended = ctx.new_activations(n, self.n_heads * self.pad, reader=self.out.reader() if plain else None)
        k.attention(q, attended, cache.k_pages, cache.v_pages, cache.page_table, ctx.row_seq, ctx.positions, self.n_heads,
                    self.n_kv_heads, self.pad, self.scale, self.window, layout=ctx, chunk=self.chunk, **ending)
        if plain:
            gated = attended
        else:
            gated = ctx.new_activations(n, self.gate_width, reader=self.out.reader())
            k.gate_heads(attended, self.pad, proj if self.gate else None, self.qkv_width, gated, self.n_heads, self.vdim,
                         **(dict(per_head=True) if self.gate_per_head else {}))
        self.out.forward(ctx, gated, out=hidden, accumulate=not fresh)
        return None

    def _queries(self, ctx, proj, cache):
        """The queries as heads of the cached size; the step's keys and values go into the cache on the way."""
        k = ctx.kernels
        if self.borrows and not cache.writes and self.rotation is None and self.pad == self.dim and proj.shape[1] == self.q_width:
            return proj      # as they were projected
        q = ctx.new_activations(ctx.n_rows, self.n_heads * self.pad)
        freq = self.rotation.frequencies(ctx.device) if self.rotation is not None else None
        turning = dict(neighbours=self.neighbours, magnitude=self.rotation.magnitude) if self.rotation is not None and (
            self.neighbours or self.rotation.magnitude != 1.0) else {}
        if self.head_norm_eps is not None and not self.head_norm_weights:
            turning["unit_norm"] = True
        if self.values_are_keys:
            turning["values_are_keys"] = True
        k.head_norm_rope_write(proj, 0, self.qkv_bias, self.q_norm, self.k_norm, self.head_norm_eps or 0.0, freq, self.turned,
                               ctx.positions, ctx.row_seq, q, cache.k_pages, cache.v_pages, cache.page_table, self.n_heads,
                               self.n_kv_heads, self.dim, self.vdim, self.pad, cache.writes, **turning)
        return q


@MIXERS.register("gated_attention")
def _build_gated_attention(config, layer_index, prefix, shared):
    sizes = config.layers[layer_index].mixer
    return GatedAttention(config.hidden, sizes.heads, sizes.kv_heads, sizes.dim, sizes.vdim, sizes.scale, prefix + "mix.",
                          bias=getattr(sizes, "bias", True), head_norm_eps=config.rms_eps, turned=sizes.rot_dims,
                          base=sizes.rot_base, chunk=getattr(sizes, "chunk", 0), window=getattr(sizes, "window", 0))


def distance_slopes(n_heads: int) -> list:
    """2^(-8 (h + 1) / n_heads) for head h: the slopes of attention with linear biases (O. Press, N. Smith, M. Lewis, "Train Short, Test
    Long: Attention with Linear Biases Enables Input Length Extrapolation")."""
    return [2.0 ** (-8.0 * (head + 1) / n_heads) for head in range(n_heads)]


@MIXERS.register("distance_attention")
def _build_distance_attention(config, layer_index, prefix, shared):
    """No rotation: a distance bias on the scores, within a window; queries that count the more the later they stand; keys and values of
    its own or another layer's."""
    sizes = config.layers[layer_index].mixer
    return GatedAttention(config.hidden, sizes.heads, sizes.kv_heads, sizes.dim, sizes.vdim, sizes.scale, prefix + "mix.", bias=False, gate=False,
                          window=sizes.window, slopes=distance_slopes(sizes.heads), q_temp=sizes.q_temp, borrows=sizes.kv_from is not None,
                          kept=config.kept_positions(layer_index))


@MIXERS.register("keyed_value_attention")
def _build_keyed_value_attention(config, layer_index, prefix, shared):
    """Values that are their keys, heads of unit root mean square, a sink of score 0, one gate a head."""
    sizes = config.layers[layer_index].mixer
    rotation = RotaryFrequencies(sizes.rot_dims, sizes.rot_base, slowed=sizes.rot_slowed) if sizes.rot_dims else None
    return GatedAttention(config.hidden, sizes.heads, sizes.kv_heads, sizes.dim, sizes.dim, sizes.scale, prefix + "mix.", bias=False,
                          head_norm_eps=config.rms_eps, head_norm_weights=False, values_are_keys=True, chunk=sizes.chunk, gate="head",
                          rotation=rotation, neighbours=True, sink=0.0)
