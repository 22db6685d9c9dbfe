"""Several agents' maps answered as one.

Every agent maps its own region (``bounding_box``); where regions overlap the reference trains one map on the other's renders
(mp_slam/mapper.py:594-706) and a point test decides which side a sample is on (mp_slam/mapper.py:491-509).  ``AgentMaps`` answers point
queries -- mesh extraction, colours of a surface, look-ups across the overlap -- from all maps at once: a point is dealt to the maps whose
boxes hold it (routing.expert_sort / expert_dispatch: each map decodes ONE contiguous run of rows), and the answers are blended
(routing.expert_combine) with weights that fall to zero where a map is left out -- at its box's faces, and where another map takes its
place among the ``top`` deepest -- so the union has no seam where a map ends."""
import torch

from .. import routing


class AgentMaps:
    """``models``: the maps (``JointEncoding`` or ``HashJointEncoding``), all on one device, this agent's own and those that
    slam_glue.load_foreign_model filled.  ``top``: of more maps that hold a point, those it is deepest in (2 by default; with 1 the deepest
    map alone answers, and there is a step where that changes)."""

    def __init__(self, models, top=2):
        self.models = list(models)
        if not self.models or top < 1:
            raise ValueError("AgentMaps needs a map and at least one choice")
        self.top = min(int(top), len(self.models))

    @torch.no_grad()
    def route(self, points):
        """``points`` [N,3] (world) -> ids [N,top] int32 (-1: no further map holds the point) and weights [N,top] float32, which add up to 1
        where any map does.  A point's weight in a map grows with its depth, the distance to the nearest face of the map's box, from
        zero at the depth of the first map that is left out (or at the face itself)."""
        boxes = torch.stack([torch.as_tensor(m.bounding_box).to(points.device, torch.float64) for m in self.models])      # [M,3,2]
        p = points.to(torch.float64)[:, None]
        depth = torch.minimum(p - boxes[..., 0], boxes[..., 1] - p).amin(-1)                                              # [N,M]
        depth, ids = torch.sort(depth, dim=1, descending=True, stable=True)
        left = depth[:, self.top:self.top + 1].clamp(min=0.0) if depth.shape[1] > self.top else 0.0
        depth, ids = depth[:, :self.top], ids[:, :self.top]
        held = depth >= 0.0                                          # (false for a point that is not a number)
        least = 1e-6 * (boxes[..., 1] - boxes[..., 0]).amin(-1)      # on a face itself, or as deep as the one left out: not zero
        w = torch.where(held, depth - left + least[ids], 0.0)
        w = w / w.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float64).tiny)
        return torch.where(held, ids, -1).to(torch.int32), w.to(torch.float32)

    @torch.no_grad()
    def query_color_sdf(self, points):
        """raw [N,4] (r, g, b logits, sdf) of points [...,3], as JointEncoding.query_color_sdf; zeros where no map holds the point."""
        flat = points.reshape(-1, 3)
        ids, weights = self.route(flat)
        plan = routing.expert_sort(ids, len(self.models))
        rows = routing.expert_dispatch(flat.to(torch.float32), plan)
        raw = torch.zeros(rows.shape[0], 4, device=rows.device)
        start = 0
        for model, size in zip(self.models, plan.sizes()):
            if size:
                raw[start:start + size] = model.query_color_sdf(rows[start:start + size])
            start += size
        return routing.expert_combine(raw, plan, weights)

    def query_sdf(self, points):
        """sdf [...] of points [...,3]; zero where no map holds the point (see ``covered``: a mesh is extracted from the points that are, or
        the edge of the union becomes a wall)."""
        return self.query_color_sdf(points)[:, 3].reshape(points.shape[:-1])

    def query_color(self, points):
        """rgb [N,3] in 0..1 of points [...,3]; grey (0.5) where no map holds the point."""
        return torch.sigmoid(self.query_color_sdf(points)[:, :3])

    def covered(self, points):
        """[...]: whether any map holds the point."""
        return (self.route(points.reshape(-1, 3))[0][:, 0] >= 0).reshape(points.shape[:-1])
