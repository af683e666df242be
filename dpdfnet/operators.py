"""Alias: `dpdfnet.operators` IS `dpdfnet_amd.operators` (same module object; see dpdfnet/__init__.py)."""
import sys as _sys

import dpdfnet_amd.operators as _m

_sys.modules[__name__] = _m
