"""Attention from one level of a point cloud to another (no counterpart in the reference, whose layers gather from a
radius only): every query point asks all key points of its cloud, whatever their number.  Used where a radius cannot
reach - a decoder's fine points asking the pooled ones, a few latent points or one token asking the whole cloud."""
import torch

from ...op_wrappers import ComputeCrossAttention, ComputeRotary
from ..cloud_ranges import CloudRanges
from .norm import LayerNormalization


class RotaryPositions(torch.nn.Module):
    """Turns pairs of a head's features by angles proportional to the point's coordinates, so that the score of a query
    and a key depends on the offset between their points.  The pairs (half of the head's features unless ``p_pairs`` says
    fewer) are dealt to the axes as evenly as they go; an axis has a geometric row of frequencies from 1 / ``p_unit`` down
    to about 1 / (``p_unit`` ``p_base``).  ``p_unit``: the length that counts as one, typically the level's cell size.
    No parameters."""

    def __init__(self, p_dims, p_head_width, p_unit=1.0, p_base=100.0, p_pairs=None, p_adjacent=False):
        super(RotaryPositions, self).__init__()
        pairs = p_head_width // 2 if p_pairs is None else int(p_pairs)
        if not 0 <= 2 * pairs <= p_head_width:
            raise RuntimeError("RotaryPositions: %d pairs in heads of %d features" % (pairs, p_head_width))
        self.num_dims_, self.head_width_, self.adjacent_ = p_dims, p_head_width, bool(p_adjacent)
        self.freqs_host_, self.axes_host_ = [], []
        for axis in range(p_dims):
            count = pairs // p_dims + (1 if axis < pairs % p_dims else 0)
            self.axes_host_ += [axis] * count
            self.freqs_host_ += [p_base ** (-j / count) / p_unit for j in range(count)]
        self.plans_ = {}                # device -> (frequencies, axes); float32 whatever type the module is moved to

    def plan(self, p_device):
        kept = self.plans_.get(p_device)
        if kept is None or kept[0].device != p_device:      # (a module that was saved elsewhere brings its tensors along)
            # whoever asks first: the plan outlives a call under inference_mode, whose tensors no training step may save
            with torch.inference_mode(False):
                self.plans_[p_device] = (torch.tensor(self.freqs_host_, dtype=torch.float32, device=p_device),
                                         torch.tensor(self.axes_host_, dtype=torch.int32, device=p_device))
        return self.plans_[p_device]

    def _apply(self, fn, *args, **kwargs):
        """Moving the module makes the plan of its new place, so that a first call within a graph's capture copies nothing
        from the host."""
        super(RotaryPositions, self)._apply(fn, *args, **kwargs)
        self.plan(fn(torch.empty(0)).device)
        return self

    def forward(self, p_feats, p_pts):
        """p_feats [N, heads, head width], p_pts float32 [N, dims]."""
        freqs, axes = self.plan(p_feats.device)
        return ComputeRotary.apply(p_feats, p_pts.contiguous(), freqs, axes, self.adjacent_)


class CrossAttention(torch.nn.Module):
    """Features of the points of ``p_pc_out`` updated from all points of the same cloud in ``p_pc_in``:

        x + proj_out(attention(rotary(proj_q(norm(x))), rotary(proj_k(norm(y))), proj_v(norm(y))))

    with x the features of the asking points [M, p_out_features] and y those of the asked ones [N, p_in_features].
    ``p_num_key_heads`` key heads are shared by groups of query heads.  Sub-modules ``norm_out_``, ``norm_in_``
    (``LayerNormalization``), ``proj_q_``, ``proj_kv_``, ``proj_out_`` (linear maps), ``rotary_``.  float32 or bfloat16
    (``.to(torch.bfloat16)``); the coordinates stay float32."""

    def __init__(self, p_dims, p_in_features, p_out_features, p_num_heads, p_head_width=None, p_num_key_heads=None,
                 p_unit=1.0):
        super(CrossAttention, self).__init__()
        heads = int(p_num_heads)
        key_heads = heads if p_num_key_heads is None else int(p_num_key_heads)
        width = p_out_features // heads if p_head_width is None else int(p_head_width)
        if heads < 1 or key_heads < 1 or heads % key_heads != 0 or width < 1:
            raise RuntimeError("CrossAttention: %d heads of %d features over %d key heads" % (heads, width, key_heads))
        self.num_heads_, self.num_key_heads_, self.head_width_ = heads, key_heads, width
        self.norm_out_, self.norm_in_ = LayerNormalization(p_out_features), LayerNormalization(p_in_features)
        self.rotary_ = RotaryPositions(p_dims, width, p_unit)
        self.proj_q_ = torch.nn.Linear(p_out_features, heads * width, bias=False)
        self.proj_kv_ = torch.nn.Linear(p_in_features, 2 * key_heads * width, bias=False)
        self.proj_out_ = torch.nn.Linear(heads * width, p_out_features)

    def forward(self, p_pc_in, p_pc_out, p_in_features, p_out_features, p_key_mask=None, p_ranges=None):
        """``p_key_mask`` bool [N]: False leaves a point of ``p_pc_in`` out.  ``p_ranges``: the two ``CloudRanges`` of
        (p_pc_in, p_pc_out) when the program keeps them (several layers of one pair of levels); without them a call makes both,
        which reads back twice and cannot be captured in a graph."""
        if p_ranges is None:
            clouds = max(p_pc_in.batch_size_host(), p_pc_out.batch_size_host())
            p_ranges = (CloudRanges(p_pc_in, clouds), CloudRanges(p_pc_out, clouds))
        asked, asking = p_ranges
        for ranges, pc, feats, which in ((asked, p_pc_in, p_in_features, "in"), (asking, p_pc_out, p_out_features, "out")):
            if not ranges.num_points_ == pc.pts_.shape[0] == feats.shape[0]:
                raise RuntimeError("CrossAttention: ranges of %d points, p_pc_%s of %d, p_%s_features of %d rows"
                                   % (ranges.num_points_, which, pc.pts_.shape[0], which, feats.shape[0]))
        queries = self.proj_q_(self.norm_out_(asking.in_order(p_out_features)))
        queries = self.rotary_(queries.reshape(-1, self.num_heads_, self.head_width_), asking.in_order(p_pc_out.pts_))
        both = self.proj_kv_(self.norm_in_(asked.in_order(p_in_features)))
        both = both.reshape(-1, 2, self.num_key_heads_, self.head_width_)
        keys = self.rotary_(both[:, 0], asked.in_order(p_pc_in.pts_))
        mask = None if p_key_mask is None else asked.in_order(p_key_mask)
        result = ComputeCrossAttention.apply(queries, keys, both[:, 1], asking.starts_, asked.starts_, asking.longest_,
                                             asked.longest_, mask, None)
        result = self.proj_out_(result.reshape(-1, self.num_heads_ * self.head_width_))
        return p_out_features + asking.back(result)
