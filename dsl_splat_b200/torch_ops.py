"""torch.ops.splat200.*: the C-ABI stages as schema'd PyTorch operators.

Each operator is the matching `stages` call (one launch sequence through
libsplat200.so on the current stream) registered with torch.library, with a
fake implementation that gives output shapes and dtypes without running the
kernels -- so the stages trace under FakeTensorMode, torch.compile and
torch.export.  The differentiable ones (`project`, `sh_forward`, `render`)
carry autograd formulas that call the backward operators, so a graph built
from them stays inside torch.ops.splat200.  The feature operators check their
arguments as `features` does, in their fake forms too.

Binning's pair count is data-dependent: its fake kernel returns an unbacked
size for point_list, which is what the reference's `.item()` read
(primitives/tiling.py:64) becomes in a traced graph.

Operator <- reference code it stands for:
  cameras_prepare     splatting/cameras.py:29-85 (camera_kernels.py:11-66)
  project             gs3d/projection.py:309-354 (tile counts for tile_mode)
  project_backward    gs3d/projection.py:357-428
  project_views       gs3d/api.py:132-189 (the per-camera projection loop, one launch)
  project_views_backward  the per-camera backward calls of that loop, summed
  sh_forward          primitives/spherical_harmonics.py:18-59 (sh.py:44-79)
  sh_backward         primitives/spherical_harmonics.py:61-101 (sh.py:82-138)
  bin_and_sort        splatting/binning.py:72-117
  render              gs3d/render.py:359-406 (features + a constant alpha channel)
  render_backward     gs3d/render.py:409-463
  rade_project        rade/projection.py:422-472 (ray planes, normals, radial depths)
  rade_project_backward  rade/projection.py:475-551
  rade_render         rade/render.py:550-601 (colour, alpha, depths, normals)
  rade_render_backward   rade/render.py:604-670
  feature_linear, feature_norm, feature_layer_norm, feature_embedding, feature_entropy
                      and their _backward: no counterpart (features.linear, .group_norm,
                      .layer_norm, .embedding, .linear_cross_entropy)
"""

from __future__ import annotations

import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import features, stages

_NS = "splat200"


def _state(centers, conics, radii, tiles, depths) -> stages.ProjectedGaussians:
    return stages.ProjectedGaussians(centers, conics, radii, tiles, depths)


# ---- cameras -------------------------------------------------------------------

@torch.library.custom_op(f"{_NS}::cameras_prepare", mutates_args=())
def cameras_prepare(views: Tensor, Ks: Tensor, width: int, height: int,
                    with_centers: bool) -> tuple[Tensor, Tensor, Tensor]:
    full, inverse, centers = stages.cameras_prepare(views, Ks, width, height, with_centers)
    return full, inverse, centers


@cameras_prepare.register_fake
def _(views, Ks, width, height, with_centers):
    count = views.numel() // 16
    full = views.new_empty(views.shape)
    inverse = views.new_empty((count if with_centers else 0, 4, 4))
    centers = views.new_empty(views.shape[:-2] + (3,) if with_centers else (0, 3))
    return full, inverse, centers


# ---- projection ----------------------------------------------------------------

@torch.library.custom_op(f"{_NS}::project", mutates_args=())
def project(means: Tensor, quats: Tensor, scales: Tensor, opacities: Tensor, view: Tensor,
            full: Tensor, K: Tensor, width: int, height: int, near: float, far: float,
            radius_clip: float, tile_mode: str) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    st = stages.project(means, quats, scales, opacities, view, full, K, width, height, near,
                        far, radius_clip, tile_mode)
    return st.centers, st.conics, st.radii, st.tile_counts, st.depths


@project.register_fake
def _(means, quats, scales, opacities, view, full, K, width, height, near, far, radius_clip,
      tile_mode):
    n = means.shape[0]
    return (means.new_empty((n, 2)), means.new_empty((n, 4)),
            means.new_empty((n,), dtype=torch.int32), means.new_empty((n,), dtype=torch.int32),
            means.new_empty((n,)))


@torch.library.custom_op(f"{_NS}::project_backward", mutates_args=())
def project_backward(means: Tensor, quats: Tensor, scales: Tensor, opacities: Tensor,
                     view: Tensor, full: Tensor, K: Tensor, width: int, height: int,
                     centers: Tensor, conics: Tensor, radii: Tensor, tiles: Tensor,
                     depths: Tensor, grad_centers: Tensor, grad_conics: Tensor
                     ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    grads = stages.project_backward(means, quats, scales, opacities, view, full, K, width, height,
                                    _state(centers, conics, radii, tiles, depths),
                                    grad_centers.contiguous(), grad_conics.contiguous(),
                                    (True,) * 6)
    # the two 4x4 camera gradients are views of one buffer: operator outputs
    # must not alias each other
    return tuple(g.clone() if i >= 4 else g for i, g in enumerate(grads))


@project_backward.register_fake
def _(means, quats, scales, opacities, view, full, K, width, height, centers, conics, radii,
      tiles, depths, grad_centers, grad_conics):
    return (torch.empty_like(means), torch.empty_like(quats), torch.empty_like(scales),
            torch.empty_like(opacities), view.new_empty((4, 4)), full.new_empty((4, 4)))


def _project_setup(ctx, inputs, output):
    means, quats, scales, opacities, view, full, K, width, height, *_ = inputs
    ctx.save_for_backward(means, quats, scales, opacities, view, full, K, *output)
    ctx.size = (width, height)


def _project_backward(ctx, g_centers, g_conics, g_radii, g_tiles, g_depths):
    means, quats, scales, opacities, view, full, K, centers, conics, radii, tiles, depths = \
        ctx.saved_tensors
    g_centers = torch.zeros_like(centers) if g_centers is None else g_centers
    g_conics = torch.zeros_like(conics) if g_conics is None else g_conics
    grads = torch.ops.splat200.project_backward(means, quats, scales, opacities, view, full, K,
                                                *ctx.size, centers, conics, radii, tiles, depths,
                                                g_centers, g_conics)
    return (*grads, None, None, None, None, None, None, None)


project.register_autograd(_project_backward, setup_context=_project_setup)


@torch.library.custom_op(f"{_NS}::project_views", mutates_args=())
def project_views(means: Tensor, quats: Tensor, scales: Tensor, opacities: Tensor,
                  views: Tensor, fulls: Tensor, Ks: Tensor, width: int, height: int, near: float,
                  far: float, radius_clip: float, sh: Tensor, sh_degree: int, campos: Tensor,
                  tile_mode: str) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """All cameras (V) of one Gaussian set in one launch (raw quaternions are
    normalised in-kernel).  Returns stacked (V, n, ...) centres, conics,
    colours, radii, tile counts, depths and the active mask."""
    out = stages.project_views(means, quats, scales, opacities, views, fulls, Ks, width, height,
                               near, far, radius_clip, sh=sh, sh_degree=sh_degree,
                               campos=campos, normalize_quats=True, tile_mode=tile_mode)
    return (torch.stack(out.centers), torch.stack(out.conics), torch.stack(out.colors),
            out.radii, out.tile_counts, out.depths, out.active)


@project_views.register_fake
def _(means, quats, scales, opacities, views, fulls, Ks, width, height, near, far, radius_clip,
      sh, sh_degree, campos, tile_mode):
    V, n = views.shape[0], means.shape[0]
    return (means.new_empty((V, n, 2)), means.new_empty((V, n, 4)), means.new_empty((V, n, 3)),
            means.new_empty((V, n), dtype=torch.int32), means.new_empty((V, n), dtype=torch.int32),
            means.new_empty((V, n)), means.new_empty((V, n, 3), dtype=torch.uint8))


@torch.library.custom_op(f"{_NS}::project_views_backward", mutates_args=())
def project_views_backward(means: Tensor, quats: Tensor, scales: Tensor, views: Tensor,
                           fulls: Tensor, Ks: Tensor, width: int, height: int, radii: Tensor,
                           sh: Tensor, sh_degree: int, campos: Tensor, active: Tensor,
                           grad_centers: Tensor, grad_conics: Tensor, grad_colors: Tensor
                           ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients of means, raw quaternions, scales, opacities and SH summed
    over the V cameras (splat_project_backward_views)."""
    V, n = views.shape[0], means.shape[0]
    outs = [torch.empty_like(t) for t in (means, quats, scales)]
    outs.append(means.new_empty(n))
    outs.append(torch.empty_like(sh))
    gc, gq, gcol = grad_centers.contiguous(), grad_conics.contiguous(), grad_colors.contiguous()
    if n and V:
        pin = stages.Args()
        from ._native import check, lib, stream
        check(lib.splat_project_backward_views(
            V, n, pin(means), None, pin(quats), pin(scales), pin(views), pin(fulls), pin(Ks),
            width, height, stages.pointer_table(radii), stages.pointer_table(gc),
            stages.pointer_table(gq), *[o.data_ptr() for o in outs[:4]], 0, sh_degree,
            sh.shape[1], pin(sh), pin(campos), stages.pointer_table(active),
            stages.pointer_table(gcol), 3, outs[4].data_ptr(), stream(means.device)),
            "project_views_backward")
    return tuple(outs)


@project_views_backward.register_fake
def _(means, quats, scales, views, fulls, Ks, width, height, radii, sh, sh_degree, campos,
      active, grad_centers, grad_conics, grad_colors):
    return (torch.empty_like(means), torch.empty_like(quats), torch.empty_like(scales),
            means.new_empty(means.shape[0]), torch.empty_like(sh))


def _project_views_setup(ctx, inputs, output):
    (means, quats, scales, opacities, views, fulls, Ks, width, height, near, far, radius_clip,
     sh, sh_degree, campos, tile_mode) = inputs
    ctx.save_for_backward(means, quats, scales, views, fulls, Ks, sh, campos, output[3],
                          output[6])
    ctx.args = (width, height, sh_degree)


def _project_views_backward(ctx, g_centers, g_conics, g_colors, *unused):
    means, quats, scales, views, fulls, Ks, sh, campos, radii, active = ctx.saved_tensors
    width, height, sh_degree = ctx.args
    V, n = views.shape[0], means.shape[0]

    def zeros(g, k):
        return means.new_zeros((V, n, k)) if g is None else g

    grads = torch.ops.splat200.project_views_backward(
        means, quats, scales, views, fulls, Ks, width, height, radii, sh, sh_degree, campos,
        active, zeros(g_centers, 2), zeros(g_conics, 4), zeros(g_colors, 3))
    gm, gq, gs, go, gsh = grads
    return (gm, gq, gs, go, None, None, None, None, None, None, None, None, gsh, None, None,
            None)


project_views.register_autograd(_project_views_backward, setup_context=_project_views_setup)


# ---- spherical harmonics ------------------------------------------------------------

@torch.library.custom_op(f"{_NS}::sh_forward", mutates_args=())
def sh_forward(coeffs: Tensor, dirs: Tensor, degree: int,
               radii: Tensor | None) -> tuple[Tensor, Tensor]:
    colors, active = stages.sh_forward(coeffs, dirs, degree, radii, True)
    return colors, active


@sh_forward.register_fake
def _(coeffs, dirs, degree, radii):
    n = coeffs.shape[0]
    return coeffs.new_empty((n, 3)), coeffs.new_empty((n, 3), dtype=torch.uint8)


@torch.library.custom_op(f"{_NS}::sh_backward", mutates_args=())
def sh_backward(coeffs: Tensor, dirs: Tensor, degree: int, radii: Tensor | None,
                active: Tensor, grad_colors: Tensor) -> tuple[Tensor, Tensor]:
    g_coeffs, g_dirs = stages.sh_backward(coeffs, dirs, degree, radii, active,
                                          grad_colors.contiguous(), True)
    return g_coeffs, g_dirs


@sh_backward.register_fake
def _(coeffs, dirs, degree, radii, active, grad_colors):
    return torch.empty_like(coeffs), dirs.new_empty((dirs.shape[0], 3))


def _sh_setup(ctx, inputs, output):
    coeffs, dirs, degree, radii = inputs
    ctx.save_for_backward(coeffs, dirs, radii, output[1])
    ctx.degree = degree


def _sh_backward(ctx, g_colors, g_active):
    coeffs, dirs, radii, active = ctx.saved_tensors
    if g_colors is None:
        return None, None, None, None
    g_coeffs, g_dirs = torch.ops.splat200.sh_backward(coeffs, dirs, ctx.degree, radii, active,
                                                      g_colors)
    return g_coeffs, g_dirs, None, None


sh_forward.register_autograd(_sh_backward, setup_context=_sh_setup)


# ---- binning -----------------------------------------------------------------------

@torch.library.custom_op(f"{_NS}::bin_and_sort", mutates_args=())
def bin_and_sort(centers: Tensor, conics: Tensor, radii: Tensor, tiles: Tensor, depths: Tensor,
                 width: int, height: int, tile_mode: str) -> tuple[Tensor, Tensor]:
    bins = stages.bin_and_sort(_state(centers, conics, radii, tiles, depths), width, height,
                               tile_mode=tile_mode)
    return bins["ranges"], bins["point_list"]


@bin_and_sort.register_fake
def _(centers, conics, radii, tiles, depths, width, height, tile_mode):
    T = ((width + 15) // 16) * ((height + 15) // 16)
    pairs = torch.library.get_ctx().new_dynamic_size()
    return (radii.new_empty((T, 2), dtype=torch.int32),
            radii.new_empty((pairs,), dtype=torch.int32))


# ---- blending ----------------------------------------------------------------------

@torch.library.custom_op(f"{_NS}::render", mutates_args=())
def render(centers: Tensor, conics: Tensor, ranges: Tensor, point_list: Tensor,
           features: Tensor, background: Tensor, width: int,
           height: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """features (N, C) blended with a constant alpha channel; background (C+1).
    Returns image (H, W, C), alpha (H, W, 1), transmittance (H, W) and
    contributor counts (H, W)."""
    out = stages.render(stages.ProjectedFootprint(centers, conics),
                        dict(ranges=ranges, point_list=point_list), features, None, True,
                        background, width, height, separate_alpha=True)
    return out.features, out.alpha, out.transmittance, out.contributors


@render.register_fake
def _(centers, conics, ranges, point_list, features, background, width, height):
    C = features.shape[1]
    return (features.new_empty((height, width, C)), features.new_empty((height, width, 1)),
            features.new_empty((height, width)),
            features.new_empty((height, width), dtype=torch.int32))


@torch.library.custom_op(f"{_NS}::render_backward", mutates_args=())
def render_backward(centers: Tensor, conics: Tensor, ranges: Tensor, point_list: Tensor,
                    features: Tensor, background: Tensor, transmittance: Tensor,
                    contributors: Tensor, grad_image: Tensor, grad_alpha: Tensor, width: int,
                    height: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of centers, conics, features and the |d centers| sums."""
    gc, gq, gf, _, gabs = stages.render_backward(
        stages.ProjectedFootprint(centers, conics), dict(ranges=ranges, point_list=point_list),
        features, None, True, background, transmittance, contributors, grad_image, width,
        height, absgrad=True, constant_tail=1, gradient_alpha=grad_alpha, separate_alpha=True,
        separate_buffers=True)
    return gc, gq, gf, gabs


@render_backward.register_fake
def _(centers, conics, ranges, point_list, features, background, transmittance, contributors,
      grad_image, grad_alpha, width, height):
    return (torch.empty_like(centers), torch.empty_like(conics), torch.empty_like(features),
            torch.empty_like(centers))


def _render_setup(ctx, inputs, output):
    centers, conics, ranges, point_list, features, background, width, height = inputs
    ctx.save_for_backward(centers, conics, ranges, point_list, features, background, output[2],
                          output[3])
    ctx.size = (width, height)


def _render_backward(ctx, g_image, g_alpha, g_t, g_contrib):
    centers, conics, ranges, point_list, features, background, final_t, contrib = \
        ctx.saved_tensors
    W, H = ctx.size
    if g_image is None:
        g_image = features.new_zeros((H, W, features.shape[1]))
    if g_alpha is None:
        g_alpha = features.new_zeros((H, W, 1))
    gc, gq, gf, _ = torch.ops.splat200.render_backward(
        centers, conics, ranges, point_list, features, background, final_t, contrib,
        g_image.contiguous(), g_alpha.contiguous(), W, H)
    return gc, gq, None, None, gf, None, None, None


render.register_autograd(_render_backward, setup_context=_render_setup)

# ---- RaDe-GS -----------------------------------------------------------------------

def _rade_config(width, height, near, far, radius_clip, kernel_size):
    from .rade.projection import ViewConfig
    return ViewConfig(width, height, near, far, radius_clip, "radius", kernel_size)


@torch.library.custom_op(f"{_NS}::rade_project", mutates_args=())
def rade_project(means: Tensor, quats: Tensor, scales: Tensor, opacities: Tensor, view: Tensor,
                 full: Tensor, K: Tensor, width: int, height: int, near: float, far: float,
                 radius_clip: float, kernel_size: float
                 ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Normalised quats.  Returns centers, conics, radii, tile counts, radial
    sort distances, ray planes and normals."""
    from .rade import projection as rp
    st = rp.prepare(means, quats, scales, opacities, view, full, K,
                    _rade_config(width, height, near, far, radius_clip, kernel_size))
    return (st.centers, st.conics, st.radii, st.tile_counts, st.depths, st.ray_planes,
            st.normals)


@rade_project.register_fake
def _(means, quats, scales, opacities, view, full, K, width, height, near, far, radius_clip,
      kernel_size):
    n = means.shape[0]
    i32 = dict(dtype=torch.int32)
    return (means.new_empty((n, 2)), means.new_empty((n, 4)), means.new_empty((n,), **i32),
            means.new_empty((n,), **i32), means.new_empty((n,)), means.new_empty((n, 3)),
            means.new_empty((n, 3)))


@torch.library.custom_op(f"{_NS}::rade_project_backward", mutates_args=())
def rade_project_backward(means: Tensor, quats: Tensor, scales: Tensor, opacities: Tensor,
                          view: Tensor, full: Tensor, K: Tensor, width: int, height: int,
                          kernel_size: float, radii: Tensor, grad_centers: Tensor,
                          grad_conics: Tensor, grad_planes: Tensor, grad_normals: Tensor
                          ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    from .rade import projection as rp
    cfg = _rade_config(width, height, 0.0, 0.0, 0.0, kernel_size)
    state = rp.ProjectedGaussians(None, None, radii, None, None, None, None)
    grads = rp.backward(means, quats, scales, opacities, view, full, K, cfg, state,
                        grad_centers.contiguous(), grad_conics.contiguous(),
                        grad_planes.contiguous(), grad_normals.contiguous(), (True,) * 6)
    # the two 4x4 camera gradients are views of one buffer: operator outputs
    # must not alias each other
    return tuple(g.clone() if i >= 4 else g for i, g in enumerate(grads[:6]))


@rade_project_backward.register_fake
def _(means, quats, scales, opacities, view, full, K, width, height, kernel_size, radii,
      grad_centers, grad_conics, grad_planes, grad_normals):
    return (torch.empty_like(means), torch.empty_like(quats), torch.empty_like(scales),
            torch.empty_like(opacities), view.new_empty((4, 4)), full.new_empty((4, 4)))


def _rade_project_setup(ctx, inputs, output):
    means, quats, scales, opacities, view, full, K, width, height, *_, kernel_size = inputs
    ctx.save_for_backward(means, quats, scales, opacities, view, full, K, output[2])
    ctx.args = (width, height, kernel_size)


def _rade_project_backward(ctx, g_centers, g_conics, g_radii, g_tiles, g_depths, g_planes,
                           g_normals):
    means, quats, scales, opacities, view, full, K, radii = ctx.saved_tensors
    n = means.shape[0]
    zero = means.new_zeros
    grads = torch.ops.splat200.rade_project_backward(
        means, quats, scales, opacities, view, full, K, *ctx.args, radii,
        zero((n, 2)) if g_centers is None else g_centers,
        zero((n, 4)) if g_conics is None else g_conics,
        zero((n, 3)) if g_planes is None else g_planes,
        zero((n, 3)) if g_normals is None else g_normals)
    return (*grads, None, None, None, None, None, None, None)


rade_project.register_autograd(_rade_project_backward, setup_context=_rade_project_setup)


@torch.library.custom_op(f"{_NS}::rade_render", mutates_args=())
def rade_render(centers: Tensor, conics: Tensor, planes: Tensor, normals: Tensor,
                ranges: Tensor, point_list: Tensor, features: Tensor, background: Tensor,
                K: Tensor, width: int, height: int
                ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """features (N, C) and background (C).  Returns the features (H, W, C),
    alpha, expected depth and median depth (H, W, 1), normals (H, W, 3),
    auxiliary (2, H, W) and contributors (2, H, W)."""
    from .rade import projection as rp
    from .rade import render as rr
    st = rp.ProjectedGaussians(centers, conics, None, None, None, planes, normals)
    out = rr.render(st, dict(ranges=ranges, point_list=point_list), features, None,
                    background, K, width, height)
    return (out.features, out.alpha, out.depth, out.median, out.normals, out.auxiliary,
            out.contributors)


@rade_render.register_fake
def _(centers, conics, planes, normals, ranges, point_list, features, background, K, width,
      height):
    C = features.shape[1]
    img = features.new_empty
    return (img((height, width, C)), img((height, width, 1)), img((height, width, 1)),
            img((height, width, 1)), img((height, width, 3)), img((2, height, width)),
            img((2, height, width), dtype=torch.int32))


@torch.library.custom_op(f"{_NS}::rade_render_backward", mutates_args=())
def rade_render_backward(centers: Tensor, conics: Tensor, planes: Tensor, normals: Tensor,
                         ranges: Tensor, point_list: Tensor, features: Tensor,
                         background: Tensor, K: Tensor, alpha: Tensor, normal_image: Tensor,
                         auxiliary: Tensor, contributors: Tensor, grad_features: Tensor,
                         grad_alpha: Tensor, grad_depth: Tensor, grad_median: Tensor,
                         grad_normals: Tensor, width: int, height: int
                         ) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    """Gradients of centers, conics, ray planes, normals, features and the
    |d centers| sums."""
    from .rade import projection as rp
    from .rade import render as rr
    st = rp.ProjectedGaussians(centers, conics, None, None, None, planes, normals)
    fwd = rr.RenderedPixels(None, alpha, None, None, normal_image, auxiliary, contributors)
    gc, gq, gf, _, gp, gn, gabs = rr.backward(
        st, dict(ranges=ranges, point_list=point_list), features, None, background, K, fwd,
        (grad_features, grad_alpha, grad_depth, grad_median, grad_normals), width, height,
        absgrad=True)
    return gc, gq, gp, gn, gf, gabs


@rade_render_backward.register_fake
def _(centers, conics, planes, normals, ranges, point_list, features, background, K, alpha,
      normal_image, auxiliary, contributors, grad_features, grad_alpha, grad_depth,
      grad_median, grad_normals, width, height):
    return (torch.empty_like(centers), torch.empty_like(conics), torch.empty_like(planes),
            torch.empty_like(normals), torch.empty_like(features), torch.empty_like(centers))


def _rade_render_setup(ctx, inputs, output):
    centers, conics, planes, normals, ranges, point_list, features, background, K, W, H = inputs
    ctx.save_for_backward(centers, conics, planes, normals, ranges, point_list, features,
                          background, K, output[1], output[4], output[5], output[6])
    ctx.size = (W, H)


def _rade_render_backward(ctx, g_feat, g_alpha, g_depth, g_median, g_normals, g_aux,
                          g_contrib):
    (centers, conics, planes, normals, ranges, point_list, features, background, K, alpha,
     normal_image, aux, contrib) = ctx.saved_tensors
    W, H = ctx.size
    zero = features.new_zeros

    def up(g, k):
        return zero((H, W, k)) if g is None else g.contiguous()

    gc, gq, gp, gn, gf, _ = torch.ops.splat200.rade_render_backward(
        centers, conics, planes, normals, ranges, point_list, features, background, K, alpha,
        normal_image, aux, contrib, up(g_feat, features.shape[1]), up(g_alpha, 1),
        up(g_depth, 1), up(g_median, 1), up(g_normals, 3), W, H)
    return gc, gq, gp, gn, None, None, gf, None, None, None, None


rade_render.register_autograd(_rade_render_backward, setup_context=_rade_render_setup)


# ---- feature operators ----------------------------------------------------------

def _check_forward_mode():
    # an operator without a formula for them drops tangents; in torch.func.jvp it
    # does not see which of its arguments had one
    if forward_ad._current_level >= 0:
        raise NotImplementedError("forward-mode derivatives of the feature operators")


def _check_linear(x, weight, bias, activation, output, name):
    _check_forward_mode()
    features.check_linear(x, weight, bias, activation, output, name)


def _check_norm(x, groups, weight, bias, eps, activation):
    _check_forward_mode()
    features._check_input(x)
    if x.ndim < 2 or x.shape[-1] < 1:
        raise ValueError("x must have samples first and at least one channel last")
    features.check_group_norm(x, groups, weight, bias, eps, activation, x.shape[0],
                              math.prod(x.shape[1:-1]))


def _check_norm_backward(x, groups, weight, bias, moments, activation, upstream):
    _check_norm(x, groups, weight, bias, 1.0, activation)
    features._check_like(upstream, x, x.shape, "upstream")
    if (moments.dtype is not torch.float32 or moments.device != x.device
            or moments.shape != (2, x.shape[0], groups)):
        raise ValueError("moments must be the float32 (2,samples,groups) of feature_norm")


@torch.library.custom_op(f"{_NS}::feature_linear", mutates_args=())
def feature_linear(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None,
                   activation: str) -> Tensor:
    _check_linear(x, weight, bias, activation, residual, "residual")
    return stages.feature_linear(x, weight, bias, residual, activation)


@feature_linear.register_fake
def _(x, weight, bias, residual, activation):
    _check_linear(x, weight, bias, activation, residual, "residual")
    return x.new_empty(x.shape[:-1] + (weight.shape[0],))


@torch.library.custom_op(f"{_NS}::feature_linear_backward", mutates_args=())
def feature_linear_backward(x: Tensor, weight: Tensor, bias: Tensor | None, activation: str,
                            upstream: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    _check_linear(x, weight, bias, activation, upstream, "upstream")
    return stages.feature_linear_backward(x, weight, bias, activation, upstream,
                                          (True, True, True))


@feature_linear_backward.register_fake
def _(x, weight, bias, activation, upstream):
    _check_linear(x, weight, bias, activation, upstream, "upstream")
    return x.new_empty(x.shape), weight.new_empty(weight.shape), x.new_empty((weight.shape[0],))


def _feature_linear_setup(ctx, inputs, output):
    x, weight, bias, residual, ctx.activation = inputs
    ctx.save_for_backward(x, weight, bias)
    ctx.with_residual = residual is not None


def _feature_linear_backward(ctx, upstream):
    x, weight, bias = ctx.saved_tensors
    dx, dw, db = torch.ops.splat200.feature_linear_backward(x, weight, bias, ctx.activation,
                                                            upstream)
    return (dx, dw, None if bias is None else db, upstream if ctx.with_residual else None, None)


feature_linear.register_autograd(_feature_linear_backward, setup_context=_feature_linear_setup)


@torch.library.custom_op(f"{_NS}::feature_norm", mutates_args=())
def feature_norm(x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None, eps: float,
                 activation: str) -> tuple[Tensor, Tensor]:
    _check_norm(x, groups, weight, bias, eps, activation)
    return stages.feature_norm(x, x.shape[0], groups, weight, bias, eps, activation)


@feature_norm.register_fake
def _(x, groups, weight, bias, eps, activation):
    _check_norm(x, groups, weight, bias, eps, activation)
    return x.new_empty(x.shape), x.new_empty((2, x.shape[0], groups), dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::feature_norm_backward", mutates_args=())
def feature_norm_backward(x: Tensor, groups: int, weight: Tensor | None, bias: Tensor | None,
                          moments: Tensor, activation: str, upstream: Tensor
                          ) -> tuple[Tensor, Tensor, Tensor]:
    _check_norm_backward(x, groups, weight, bias, moments, activation, upstream)
    return stages.feature_norm_backward(x, x.shape[0], groups, weight, bias, moments, activation,
                                        upstream, (True, True, True))


@feature_norm_backward.register_fake
def _(x, groups, weight, bias, moments, activation, upstream):
    _check_norm_backward(x, groups, weight, bias, moments, activation, upstream)
    return (x.new_empty(x.shape), x.new_empty((x.shape[-1],)), x.new_empty((x.shape[-1],)))


def _feature_norm_setup(ctx, inputs, output):
    x, ctx.groups, weight, bias, _eps, ctx.activation = inputs
    ctx.save_for_backward(x, weight, bias, output[1])


def _feature_norm_backward(ctx, upstream, _moments):
    x, weight, bias, moments = ctx.saved_tensors
    dx, dw, db = torch.ops.splat200.feature_norm_backward(x, ctx.groups, weight, bias, moments,
                                                          ctx.activation, upstream)
    return (dx, None, None if weight is None else dw, None if bias is None else db, None, None)


feature_norm.register_autograd(_feature_norm_backward, setup_context=_feature_norm_setup)


def _check_layer_norm(x, weight, bias, eps, activation, upstream=None):
    _check_forward_mode()
    features.check_layer_norm(x, weight, bias, eps, activation)
    features._check_like(upstream, x, x.shape, "upstream")


@torch.library.custom_op(f"{_NS}::feature_layer_norm", mutates_args=())
def feature_layer_norm(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
                       activation: str) -> Tensor:
    _check_layer_norm(x, weight, bias, eps, activation)
    return stages.feature_layer_norm(x, weight, bias, eps, activation)


@feature_layer_norm.register_fake
def _(x, weight, bias, eps, activation):
    _check_layer_norm(x, weight, bias, eps, activation)
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{_NS}::feature_layer_norm_backward", mutates_args=())
def feature_layer_norm_backward(x: Tensor, weight: Tensor | None, bias: Tensor | None, eps: float,
                                activation: str, upstream: Tensor
                                ) -> tuple[Tensor, Tensor, Tensor]:
    _check_layer_norm(x, weight, bias, eps, activation, upstream)
    return stages.feature_layer_norm_backward(x, weight, bias, eps, activation, upstream,
                                              (True, True, True))


@feature_layer_norm_backward.register_fake
def _(x, weight, bias, eps, activation, upstream):
    _check_layer_norm(x, weight, bias, eps, activation, upstream)
    return (x.new_empty(x.shape), x.new_empty((x.shape[-1],)), x.new_empty((x.shape[-1],)))


def _feature_layer_norm_setup(ctx, inputs, output):
    x, weight, bias, *ctx.settings = inputs
    ctx.save_for_backward(x, weight, bias)


def _feature_layer_norm_backward(ctx, upstream):
    x, weight, bias = ctx.saved_tensors
    dx, dw, db = torch.ops.splat200.feature_layer_norm_backward(x, weight, bias, *ctx.settings,
                                                                upstream)
    return dx, None if weight is None else dw, None if bias is None else db, None, None


feature_layer_norm.register_autograd(_feature_layer_norm_backward,
                                     setup_context=_feature_layer_norm_setup)


def _check_embedding(ids, table, scale):
    _check_forward_mode()
    if table.ndim != 2:
        raise ValueError("table must be (V,C) with V and C of at least one")
    features.check_embedding(ids, table.shape[0], table.shape[1], scale, table)


def _check_embedding_backward(ids, entries, scale, upstream):
    _check_forward_mode()
    if upstream.ndim != ids.ndim + 1 or upstream.shape[:-1] != ids.shape:
        raise ValueError("upstream must have the shape of ids and channels last")
    features.check_embedding(ids, entries, upstream.shape[-1], scale, upstream)


@torch.library.custom_op(f"{_NS}::feature_embedding", mutates_args=())
def feature_embedding(ids: Tensor, table: Tensor, scale: float) -> Tensor:
    _check_embedding(ids, table, scale)
    return stages.feature_embedding(ids, table, scale)


@feature_embedding.register_fake
def _(ids, table, scale):
    _check_embedding(ids, table, scale)
    return table.new_empty(ids.shape + (table.shape[1],))


@torch.library.custom_op(f"{_NS}::feature_embedding_backward", mutates_args=())
def feature_embedding_backward(ids: Tensor, entries: int, scale: float,
                               upstream: Tensor) -> Tensor:
    _check_embedding_backward(ids, entries, scale, upstream)
    return stages.feature_embedding_backward(ids, entries, scale, upstream)


@feature_embedding_backward.register_fake
def _(ids, entries, scale, upstream):
    _check_embedding_backward(ids, entries, scale, upstream)
    return upstream.new_empty((entries, upstream.shape[-1]))


def _feature_embedding_setup(ctx, inputs, output):
    ids, table, ctx.scale = inputs
    ctx.save_for_backward(ids)
    ctx.entries = table.shape[0]


def _feature_embedding_backward(ctx, upstream):
    ids, = ctx.saved_tensors
    return None, torch.ops.splat200.feature_embedding_backward(ids, ctx.entries, ctx.scale,
                                                               upstream), None


feature_embedding.register_autograd(_feature_embedding_backward,
                                    setup_context=_feature_embedding_setup)


def _check_entropy(x, weight, target, bias, ignore_index, reduction):
    _check_forward_mode()
    features.check_linear_cross_entropy(x, weight, target, bias, ignore_index, reduction)


def _check_entropy_backward(x, weight, target, bias, ignore_index, reduction, moments, counted,
                            upstream):
    _check_entropy(x, weight, target, bias, ignore_index, reduction)
    upstream_shape = target.shape if reduction == "none" else ()
    for t, shape, name in ((moments, (target.numel(), 2), "moments"), (counted, (1,), "counted"),
                           (upstream, upstream_shape, "upstream")):
        if t.dtype is not torch.float32 or t.device != x.device or t.shape != shape:
            raise ValueError(f"{name} must be float32 of shape {tuple(shape)} on x's device")


@torch.library.custom_op(f"{_NS}::feature_entropy", mutates_args=())
def feature_entropy(x: Tensor, weight: Tensor, target: Tensor, bias: Tensor | None,
                    ignore_index: int, reduction: str) -> tuple[Tensor, Tensor, Tensor]:
    _check_entropy(x, weight, target, bias, ignore_index, reduction)
    return stages.feature_entropy(x, weight, target, bias, ignore_index, reduction)


@feature_entropy.register_fake
def _(x, weight, target, bias, ignore_index, reduction):
    _check_entropy(x, weight, target, bias, ignore_index, reduction)
    f32 = torch.float32
    return (x.new_empty(target.shape if reduction == "none" else (), dtype=f32),
            x.new_empty((target.numel(), 2), dtype=f32), x.new_empty((1,), dtype=f32))


@torch.library.custom_op(f"{_NS}::feature_entropy_backward", mutates_args=())
def feature_entropy_backward(x: Tensor, weight: Tensor, target: Tensor, bias: Tensor | None,
                             ignore_index: int, reduction: str, moments: Tensor, counted: Tensor,
                             upstream: Tensor) -> tuple[Tensor, Tensor, Tensor]:
    _check_entropy_backward(x, weight, target, bias, ignore_index, reduction, moments, counted,
                            upstream)
    dx, dweight, dbias = stages.feature_entropy_backward(
        x, weight, target, bias, ignore_index, reduction, moments, counted, upstream,
        (True, True, True))
    return dx, dweight, weight.new_empty((0,)) if dbias is None else dbias


@feature_entropy_backward.register_fake
def _(x, weight, target, bias, ignore_index, reduction, moments, counted, upstream):
    _check_entropy_backward(x, weight, target, bias, ignore_index, reduction, moments, counted,
                            upstream)
    return (x.new_empty(x.shape), weight.new_empty(weight.shape),
            weight.new_empty((0 if bias is None else weight.shape[0],)))


def _feature_entropy_setup(ctx, inputs, output):
    x, weight, target, bias, *ctx.settings = inputs
    ctx.save_for_backward(x, weight, target, bias, output[1], output[2])


def _feature_entropy_backward(ctx, upstream, _moments, _counted):
    x, weight, target, bias, moments, counted = ctx.saved_tensors
    dx, dw, db = torch.ops.splat200.feature_entropy_backward(
        x, weight, target, bias, *ctx.settings, moments, counted, upstream)
    return dx, dw, None, None if bias is None else db, None, None


feature_entropy.register_autograd(_feature_entropy_backward,
                                  setup_context=_feature_entropy_setup)

OPERATORS = ("cameras_prepare", "project", "project_backward", "project_views",
             "project_views_backward", "sh_forward", "sh_backward", "bin_and_sort", "render",
             "render_backward", "rade_project", "rade_project_backward", "rade_render",
             "rade_render_backward", "feature_linear", "feature_linear_backward", "feature_norm",
             "feature_norm_backward", "feature_layer_norm", "feature_layer_norm_backward",
             "feature_embedding", "feature_embedding_backward", "feature_entropy",
             "feature_entropy_backward")
