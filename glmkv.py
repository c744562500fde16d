"""`import glmkv` with this directory on the path: the package lies in kern-glm53_b200/, and this module puts it
in its own place. With kern-glm53_b200/ first on the path the package is found there and this file is not read."""
import importlib.util
import pathlib
import sys

_init = pathlib.Path(__file__).resolve().parent / "kern-glm53_b200" / "glmkv" / "__init__.py"
_spec = importlib.util.spec_from_file_location(__name__, _init, submodule_search_locations=[str(_init.parent)])
_package = importlib.util.module_from_spec(_spec)
sys.modules[__name__] = _package
_spec.loader.exec_module(_package)
