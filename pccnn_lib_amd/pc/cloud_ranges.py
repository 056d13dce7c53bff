import torch


class CloudRanges(object):
    """Where the clouds of a batch lie when they are stored one behind the other - what ``cross_attention`` takes beside
    its features (no counterpart in the reference): ``starts_`` int32 [clouds + 1] on the device, ``longest_`` (the largest
    cloud's points, an int) and, for a batch whose points are not in cloud order, ``order_`` (int64 [N], the points sorted
    by cloud, else None).  Built once per level with one read-back; ``p_batch_size`` makes room for clouds without points
    at the end of the batch."""

    def __init__(self, p_pc, p_batch_size=None):
        ids = p_pc.batch_ids_
        clouds = p_pc.batch_size_host() if p_batch_size is None else int(p_batch_size)
        if clouds < p_pc.batch_size_host():
            raise RuntimeError("CloudRanges: %d clouds, but the batch ids go up to %d"
                               % (clouds, p_pc.batch_size_host() - 1))
        with torch.inference_mode(False), torch.no_grad():      # kept by programs that serve first and train later
            counts = torch.bincount(ids.to(torch.int64), minlength=clouds)
            starts = torch.zeros((clouds + 1,), dtype=torch.int64, device=ids.device)
            torch.cumsum(counts, 0, out=starts[1:])
            self.starts_ = starts.to(torch.int32)
            out_of_order = (ids[1:] < ids[:-1]).sum()
            longest, out_of_order = torch.stack([counts.max(), out_of_order]).tolist()
            self.longest_ = int(longest)
            self.num_points_ = ids.shape[0]
            self.order_ = self.inverse_ = None
            if out_of_order:
                self.order_ = torch.argsort(ids, stable=True)
                self.inverse_ = torch.empty_like(self.order_)
                self.inverse_[self.order_] = torch.arange(ids.shape[0], device=ids.device)

    def in_order(self, p_rows):
        """Per-point rows in cloud order (the tensor itself when the batch is stored that way)."""
        return p_rows if self.order_ is None else torch.index_select(p_rows, 0, self.order_)

    def back(self, p_rows):
        """Rows in cloud order, back in the batch's own order."""
        return p_rows if self.inverse_ is None else torch.index_select(p_rows, 0, self.inverse_)
