from .module import Int8WideMLP, WideMLP

__all__ = ["Int8WideMLP", "WideMLP"]
