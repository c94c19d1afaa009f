from .cache import PageCache, PageCacheConfig, PageCacheView, PageMetadata, build_query_start_loc, build_tree_mask

__all__ = ("PageCache", "PageCacheConfig", "PageCacheView", "PageMetadata", "build_query_start_loc", "build_tree_mask")
